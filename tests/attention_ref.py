"""64-bit reference of the block-sparse attention and its error bounds.

The bounds follow the kernels' roundings, each off by at most u = eps / 2 of
the type relative to the value: results are rounded to the type (u), and so are
the probabilities and the score gradients before their products (u).  What is
kept in fp32 (scores, exponentials, sums) adds less than C = 2^-13 relative to
the sum of magnitudes: a product of dim <= 128 terms in fp32 is off by
128 * 2^-24 of that sum, and with scores below 64 an exponential by 64 * 2^-24 times
a few.
"""
import math

import torch

C = 2.0 ** -13


def pairs(blocks, nblocks, q_len, k_len, block, causal, ql, kl):
    """(k_heads, q_len, k_len) of one batch element: who reads whom; and positions."""
    on = torch.zeros(blocks.shape[0], q_len, nblocks + 1, dtype=torch.bool, device=blocks.device)
    on.scatter_(2, torch.where((blocks >= 0) & (blocks < nblocks), blocks, nblocks).long(), True)
    on = on[..., :nblocks].repeat_interleave(block, 2)[..., :k_len]
    p = torch.arange(q_len, device=blocks.device) + kl - ql
    j = torch.arange(k_len, device=blocks.device)
    ok = (j < kl) & (torch.arange(q_len, device=blocks.device) < ql)[:, None]
    if causal:
        ok = ok & (j <= p[:, None])
    return on & ok, p


def attention(q, k, v, blocks, block, causal, scale, q_lens, k_lens, table=None, edges=None, dout=None):
    """Results and the bounds of their errors, by name.  Entries behind a sequence's end are 0 (lse: -inf)."""
    B, n, hq, d = q.shape
    nk, hkv = k.shape[1:3]
    g = hq // hkv
    u = torch.finfo(q.dtype).eps / 2
    nb = -(-nk // block)
    f8, dev = torch.float64, q.device
    z = lambda *s: torch.zeros(*s, dtype=f8, device=dev)  # noqa: E731
    r = {"out": z(B, n, hq, d), "lse": torch.full((B, hq, n), -math.inf, dtype=f8, device=dev)}
    e = {"out": z(B, n, hq, d), "lse": z(B, hq, n)}
    if dout is not None:
        for x in (r, e):
            x.update(dq=z(B, n, hq, d), dk=z(B, nk, hkv, d), dv=z(B, nk, hkv, d))
            if table is not None:
                x["dtable"] = z(*table.shape)
    for b in range(B):
        ql = n if q_lens is None else int(q_lens[b])
        kl = nk if k_lens is None else int(k_lens[b])
        ok, p = pairs(blocks[b], nb, n, nk, block, causal, ql, kl)
        bucket = None
        if table is not None:
            dist = torch.arange(nk, device=dev) - p[:, None]
            bucket = (edges.long()[:, None, None] <= dist).sum(0)
        for h in range(hq):
            m = ok[h // g]
            row, col = m.any(1), m.any(0)
            Q = torch.where(row[:, None], q[b, :, h], 0).to(f8)
            K = torch.where(col[:, None], k[b, :, h // g], 0).to(f8)
            V = torch.where(col[:, None], v[b, :, h // g], 0).to(f8)
            x = Q @ K.t() * scale
            if table is not None:
                x = x + table[:, h].to(f8)[bucket]
            x = torch.where(m, x, -math.inf)
            top = torch.where(row, x.amax(1), 0.0)[:, None]
            w = (x - top).exp()
            total = w.sum(1, keepdim=True)
            P = w / torch.where(total > 0, total, 1.0)
            O = P @ V
            Oe = u * O.abs() + (u + C) * (P @ V.abs())
            r["out"][b, :, h], e["out"][b, :, h] = O, Oe
            lse = torch.where(row, top[:, 0] + total[:, 0].log(), -math.inf)
            r["lse"][b, h], e["lse"][b, h] = lse, torch.where(row, C / 8 * (1 + lse.abs()), 0.0)
            if dout is None:
                continue
            D = torch.where(row[:, None], dout[b, :, h], 0).to(f8)
            dP = D @ V.t()
            delta = (D * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            # delta is taken from the rounded out
            off = (D.abs() * Oe).sum(1, keepdim=True)
            E = P * (off + (u + C) * (dP.abs() + delta.abs()) + C / 16 * (D.abs() @ V.abs().t()))
            dq = dS @ K * scale
            r["dq"][b, :, h], e["dq"][b, :, h] = dq, E @ K.abs() * abs(scale) + u * dq.abs()
            r["dk"][b, :, h // g] += dS.t() @ Q * scale
            e["dk"][b, :, h // g] += E.t() @ Q.abs() * abs(scale)
            r["dv"][b, :, h // g] += P.t() @ D
            e["dv"][b, :, h // g] += (u + C) * (P.t() @ D.abs())
            if table is not None:
                for t in range(table.shape[0]):
                    at = bucket == t
                    r["dtable"][t, h] += dS[at].sum()
                    e["dtable"][t, h] += E[at].sum()
    for name in ("dk", "dv", "dtable"):
        if name in r:
            e[name] += u * r[name].abs()
    # the smallest numbers of the type are further apart than u times themselves
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for name in e:
        e[name] += tiny if name != "lse" else 1e-6
    return r, e


def select(q, summary, keep, k_len, block, causal, first, local, q_lens, k_lens):
    """The pattern by the definition, one query at a time on the host."""
    B, n, hq, d = q.shape
    hkv, m = summary.shape[1:3]
    g = hq // hkv
    got = torch.full((B, hkv, n, keep), -1, dtype=torch.int32)
    s = torch.stack([(q[:, :, h].double().cpu()[:, :, None] * summary[:, h // g].double().cpu()[:, None]).sum(3)
                     for h in range(hq)], 1)
    s = torch.where(s.isnan(), -math.inf, s).view(B, hkv, g, n, m).amax(2)
    for b in range(B):
        ql = n if q_lens is None else int(q_lens[b])
        kl = k_len if k_lens is None else int(k_lens[b])
        for i in range(ql):
            p = i + kl - ql
            seen = (p // block + 1 if p >= 0 else 0) if causal else -(-kl // block)
            must = list(range(min(first, seen)))
            if causal:
                must += [c for c in range(max(0, seen - local), seen) if c not in must]
            for h in range(hkv):
                rest = [c for c in range(seen) if c not in must]
                rest.sort(key=lambda c: (-float(s[b, h, i, c]), c))
                row = sorted((must + rest)[:keep])
                got[b, h, i, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return got
