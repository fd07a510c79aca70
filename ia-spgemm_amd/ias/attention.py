"""Block-sparse attention and the relative position bias on torch tensors
(the ias_block_* and ias_rel_bias* entry points of include/ias.h).

q is (batch, q_len, q_heads, dim), k and v are (batch, k_len, k_heads, dim),
bf16 or fp16 on one HIP device; any strides whose last is 1 and whose others
are multiples of 8.  Calls enqueue work on the current stream of the tensors'
device and return without waiting; outputs and workspaces come from torch's
allocator on that stream, so the calls can be captured into a graph.

    m      = block_summary(k)
    blocks = block_select(q, m, keep=16, k_len=k.shape[1])
    out, lse = block_attention(q, k, v, blocks)
    dq, dk, dv, _ = block_attention_grad(dout, q, k, v, out, lse, blocks)

There is no autograd function here: the gradient is a call of its own.  A call whose
tensors require a gradient is refused where torch records (its results would be without
one and nobody would notice): call it under torch.no_grad(), in an autograd function of
yours, or on detached tensors.  block_select takes any, since a pattern has no gradient.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import Attention, Heads, check, lib

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _no_graph(**tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} requires a gradient, and this call records none: use torch.no_grad() and the "
                                 "gradient's own call")


def _written(t: torch.Tensor) -> None:
    """Tells torch of a write through an address."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _device(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("ias.attention takes tensors of a HIP device")
    return t.device.index


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _heads(t: torch.Tensor, shape, dtype, device, name: str) -> Heads:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, not {dtype} {tuple(shape)} on {device}")
    s = t.stride()
    if s[3] != 1 and t.numel():
        raise ValueError(f"{name}: the last dimension has to be contiguous")
    return Heads(t.data_ptr(), s[0], s[1], s[2])


def _plain(t: Optional[torch.Tensor], shape, dtype, device, name: str) -> Optional[int]:
    """Address of a contiguous tensor of that shape and type."""
    if t is None:
        return None
    if not t.is_contiguous() or t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} has to be a contiguous {dtype} {tuple(shape)} on {device}, not {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _attention(like: torch.Tensor, batch, q_len, k_len, q_heads, k_heads, dim, block, keep, causal, scale, q_lens,
               k_lens, table=None, edges=None) -> Attention:
    device, dtype = _device(like), _DTYPE.get(like.dtype)
    if dtype is None:
        raise ValueError(f"{like.dtype} is not supported")
    a = Attention(dtype, device, _stream(device), batch, q_len, k_len, q_heads, k_heads, dim, block, keep, 1 if causal else 0,
                  float(scale) if scale is not None else (dim ** -0.5 if dim else 1.0), 0,
                  None if q_lens is None else _plain(q_lens, (batch,), torch.int32, like.device, "q_lens"),
                  None if k_lens is None else _plain(k_lens, (batch,), torch.int32, like.device, "k_lens"))
    if (table is None) != (edges is None):
        raise ValueError("table and edges go together")
    if table is not None:
        a.num_buckets = table.shape[0]
        a.table = _plain(table, (edges.numel() + 1, q_heads), like.dtype, like.device, "table")
        a.edges = _plain(edges, (table.shape[0] - 1,), torch.int32, like.device, "edges")
        if table.shape[0] == 1:
            a.edges = a.table  # no edge to read
    return a


def _new(shape, dtype, device):
    """A tensor and its description."""
    t = torch.empty(shape, dtype=dtype, device=device)
    _, n, h, d = shape
    return t, Heads(t.data_ptr(), n * h * d, h * d, d)


def block_summary(k: torch.Tensor, *, block: int = 64, k_lens: Optional[torch.Tensor] = None, fresh: int = 0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(batch, k_heads, blocks, dim): the mean of each block of keys.  With
    `fresh`, `out` is the summary of a cache that has grown by that many tokens
    since: only the blocks that hold them are written."""
    b, n, h, d = k.shape
    if fresh and out is None:
        raise ValueError("fresh brings an existing summary up to date: pass it as out")
    _no_graph(k=k, out=out)
    a = _attention(k, b, 0, n, h, h, d, block, 1, True, None, None, k_lens)
    shape = (b, h, -(-n // block) if block > 0 else 0, d)
    given = out is not None
    if not given:
        out = torch.empty(shape, dtype=k.dtype, device=k.device)
    check(lib.ias_block_summary(C.byref(a), C.byref(_heads(k, k.shape, k.dtype, k.device, "k")), fresh,
                                _plain(out, shape, k.dtype, k.device, "out")), "ias_block_summary")
    if given:
        _written(out)
    return out


def block_select(q: torch.Tensor, summary: torch.Tensor, keep: int, *, k_len: int, block: int = 64, causal: bool = True,
                 first: int = 1, local: int = 1, q_lens: Optional[torch.Tensor] = None,
                 k_lens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(batch, k_heads, q_len, keep) int32: the blocks that each query reads,
    ascending, -1 behind.  `first` blocks and (causal) the `local` last ones
    always, then those whose summary scores highest."""
    b, n, hq, d = q.shape
    a = _attention(q, b, n, k_len, hq, summary.shape[1], d, block, keep, causal, None, q_lens, k_lens)
    m = -(-k_len // block) if block > 0 else 0
    given = out is not None
    if not given:
        out = torch.empty((b, summary.shape[1], n, max(keep, 0)), dtype=torch.int32, device=q.device)
        a.clear = 1
    check(lib.ias_block_select(C.byref(a), C.byref(_heads(q, q.shape, q.dtype, q.device, "q")),
                               _plain(summary, (b, summary.shape[1], m, d), q.dtype, q.device, "summary"), first,
                               local if causal else 0,
                               _plain(out, (b, summary.shape[1], n, keep), torch.int32, q.device, "out")),
          "ias_block_select")
    if given:
        _written(out)
    return out


def _shapes(q, k, blocks, block, causal, scale, q_lens, k_lens, table, edges):
    b, n, hq, d = q.shape
    nk, hkv = k.shape[1], k.shape[2]
    a = _attention(q, b, n, nk, hq, hkv, d, block, blocks.shape[-1], causal, scale, q_lens, k_lens, table, edges)
    return a, (b, n, hq, d), (b, nk, hkv, d), _plain(blocks, (b, hkv, n, blocks.shape[-1]), torch.int32, q.device, "blocks")


def _workspace(pa, device, backward: bool):
    n = C.c_int64(0)
    check(lib.ias_block_attention_workspace(pa, None if backward else C.byref(n), C.byref(n) if backward else None),
          "ias_block_attention_workspace")
    return (torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None), n.value


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor, *, block: int = 64,
                    causal: bool = True, scale: Optional[float] = None, q_lens: Optional[torch.Tensor] = None,
                    k_lens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None,
                    edges: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, lse): softmax(scale q k^T + bias) v over the pattern, and the
    logarithm of each row's sum, (batch, q_heads, q_len) in fp32.  Rows behind
    q_lens are 0 / -inf in new tensors and left alone in a given `out`."""
    _no_graph(q=q, k=k, v=v, table=table, out=out)
    a, qs, ks, pb = _shapes(q, k, blocks, block, causal, scale, q_lens, k_lens, table, edges)
    dtype, device = q.dtype, q.device
    if out is None:
        out, ho = _new(qs, dtype, device)
        a.clear = 1
    else:
        ho = _heads(out, qs, dtype, device, "out")
    lse = torch.empty((qs[0], qs[2], qs[1]), dtype=torch.float32, device=device)
    if not a.clear and q_lens is not None:
        lse.fill_(float("-inf"))
    pa = C.byref(a)
    ws, n = _workspace(pa, device, False)
    check(lib.ias_block_attention(pa, C.byref(_heads(q, qs, dtype, device, "q")), C.byref(_heads(k, ks, dtype, device, "k")),
                                  C.byref(_heads(v, ks, dtype, device, "v")), pb, C.byref(ho), lse.data_ptr(), _address(ws), n),
          "ias_block_attention")
    if not a.clear:
        _written(out)
    return out, lse


def block_attention_grad(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                         lse: torch.Tensor, blocks: torch.Tensor, *, block: int = 64, causal: bool = True,
                         scale: Optional[float] = None, q_lens: Optional[torch.Tensor] = None,
                         k_lens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None,
                         edges: Optional[torch.Tensor] = None):
    """(dq, dk, dv, dtable) from the forward call's arguments and results;
    dtable is None without a table."""
    _no_graph(dout=dout, q=q, k=k, v=v, out=out, lse=lse, table=table)
    a, qs, ks, pb = _shapes(q, k, blocks, block, causal, scale, q_lens, k_lens, table, edges)
    dtype, device = q.dtype, q.device
    (dq, hq), (dk, hk), (dv, hv) = _new(qs, dtype, device), _new(ks, dtype, device), _new(ks, dtype, device)
    a.clear = 1
    dtable = None if table is None else torch.empty_like(table)
    pl = _plain(lse, (qs[0], qs[2], qs[1]), torch.float32, device, "lse")
    pa = C.byref(a)
    ws, n = _workspace(pa, device, True)
    p = [C.byref(_heads(t, s, dtype, device, x)) for t, s, x in (
        (dout, qs, "dout"), (q, qs, "q"), (k, ks, "k"), (v, ks, "v"), (out, qs, "out"))]
    check(lib.ias_block_attention_grad(pa, p[0], p[1], p[2], p[3], p[4], pl, pb, C.byref(hq), C.byref(hk), C.byref(hv),
                                       _address(dtable), _address(ws), n),
          "ias_block_attention_grad")
    return dq, dk, dv, dtable


def rel_bias(table: torch.Tensor, edges: torch.Tensor, q_len: int, k_len: int) -> torch.Tensor:
    """(heads, q_len, k_len): table[bucket(j - i - (k_len - q_len)), h], where
    bucket(d) is how many of the ascending `edges` are <= d."""
    _no_graph(table=table)
    device = _device(table)
    if table.dtype not in _DTYPE:
        raise ValueError(f"{table.dtype} is not supported")
    pt = _plain(table, (edges.numel() + 1, table.shape[1]), table.dtype, table.device, "table")
    pe = _plain(edges, (edges.numel(),), torch.int32, table.device, "edges") or pt
    out = torch.empty((table.shape[1], q_len, k_len), dtype=table.dtype, device=table.device)
    check(lib.ias_rel_bias(_DTYPE[table.dtype], table.shape[1], q_len, k_len, table.shape[0], pt, pe, out.data_ptr(),
                           device, _stream(device)), "ias_rel_bias")
    return out


def rel_bias_grad(grad: torch.Tensor, edges: torch.Tensor) -> torch.Tensor:
    """(buckets, heads) of grad's type: the sum of grad (batch, heads, q_len,
    k_len) over each bucket of each head."""
    _no_graph(grad=grad)
    device = _device(grad)
    if grad.dtype not in _DTYPE or grad.dim() != 4:
        raise ValueError(f"grad: {grad.dtype} {tuple(grad.shape)} is not supported")
    b, h, n, m = grad.shape
    if grad.numel() and m > 1 and grad.stride(3) != 1:
        raise ValueError("grad: the last dimension has to be contiguous")
    pe = _plain(edges, (edges.numel(),), torch.int32, grad.device, "edges")
    buckets = edges.numel() + 1
    out = torch.empty((buckets, h), dtype=grad.dtype, device=grad.device)
    need = C.c_int64(0)
    check(lib.ias_rel_bias_grad_workspace(b, h, n, m, buckets, C.byref(need)), "ias_rel_bias_grad_workspace")
    ws = torch.empty(need.value, dtype=torch.uint8, device=grad.device)
    check(lib.ias_rel_bias_grad(_DTYPE[grad.dtype], b, h, n, m, buckets, grad.data_ptr(), grad.stride(0), grad.stride(1),
                                grad.stride(2), pe or out.data_ptr(), out.data_ptr(), ws.data_ptr(), need.value, device,
                                _stream(device)), "ias_rel_bias_grad")
    return out
