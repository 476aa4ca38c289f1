"""Masked attention in 64 bits, with a bound for each output that the kernels' roundings cannot pass.

u = half a step of the type that P, dS and the outputs are rounded to (bf16 2^-8, fp32 2^-24).  A score is off by at most
  es = (D + 8) 2^-24 (|q| . |k|) scale + 2^-20 cap     (sums in 32 bits; the cap's tanh is within 2^-20)
     + 2^-22 (|s| + slope distance)
and a probability by the factor ep = 2 max_row es + 2^-20 (its own score, the log-sum-exp, the exponential).  Sums over n
terms in 32 bits add n 2^-24 of the sum of absolute values.  Every bound below is a sum of such terms, computed with the
absolute values in place of the values.
"""
import torch


def ranges_of(batch, seq_q, seq_kv, causal=False, starts=None, prefixes=None, offset=0):
    """The definition, position by position."""
    out = torch.zeros((batch, seq_q, 2), dtype=torch.int32)
    for b in range(batch):
        for i in range(seq_q):
            p, lo, end, prefix = offset + i, 0, seq_kv, 0
            if starts is not None:
                lo = end = -1
                for d in range(starts.shape[1] - 1):
                    if starts[b, d] <= p < starts[b, d + 1]:
                        lo, end = int(starts[b, d]), int(starts[b, d + 1])
                        prefix = int(prefixes[b, d]) if prefixes is not None else 0
                if lo < 0:
                    continue
            elif prefixes is not None:
                prefix = int(prefixes[b, 0])
            end = min(end, seq_kv)
            hi = min(end, max(p + 1, lo + max(prefix, 0))) if causal else end
            if lo < hi:
                out[b, i, 0], out[b, i, 1] = lo, hi
    return out


def attention(q, k, v, scale, causal=False, cap=0.0, ranges=None, slopes=None, offset=0, d_o=None, unit=2.0 ** -24):
    """dict of o, lse (and dq, dk, dv), and of the bounds under the same names with "_tol" behind; all on the CPU, from
    tensors of any type [B, S, heads, D]."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, Sq, H, D = q.shape
    Skv, KH = k.shape[1], k.shape[2]
    G = H // KH
    i, j = torch.arange(Sq)[:, None], torch.arange(Skv)[None, :]
    seen = torch.ones((B, Sq, Skv), dtype=torch.bool)
    if ranges is not None:
        r = ranges.cpu().long()
        seen = (j >= r[..., :1]) & (j < r[..., 1:])
    if causal:
        seen = seen & (j <= i + offset)
    seen = seen[:, None].expand(B, H, Sq, Skv)

    def heads(t):
        t = t.permute(0, 2, 1, 3)
        return t if t.shape[1] == H else t.repeat_interleave(G, dim=1)

    # rows and keys that nobody sees may hold anything
    row_used, key_used = seen[:, 0].any(dim=2), seen[:, 0].any(dim=1)
    Q = torch.where(row_used[:, None, :, None], heads(q), 0.0)
    K, V = (torch.where(key_used[:, None, :, None], heads(t), 0.0) for t in (k, v))
    x = Q @ K.transpose(2, 3) * scale
    size = Q.abs() @ K.abs().transpose(2, 3) * scale
    t = torch.tanh(x / cap) if cap else None
    s = cap * t if cap else x
    far = torch.zeros_like(s)
    if slopes is not None:
        far = slopes.detach().cpu().double()[None, :, None, None] * (i + offset - j).abs().double()
        s = s - far
    e32 = 2.0 ** -24
    es = (D + 8) * e32 * size + 4 * e32 * (s.abs() + far) + 16 * e32 * cap
    es = torch.where(seen, es, 0.0).amax(dim=3, keepdim=True)
    s = torch.where(seen, s, float("-inf"))
    lse = torch.logsumexp(s, dim=3)
    empty = lse == float("-inf")
    p = torch.exp(s - torch.where(empty, 0.0, lse)[..., None])
    ep = 2 * es + 16 * e32
    pv = p @ V.abs()
    o = p @ V
    o_tol = (unit + ep + (Skv + 16) * e32) * pv + unit * o.abs()
    back = lambda a: a.permute(0, 2, 1, 3).contiguous()  # noqa: E731
    out = {"o": back(o), "o_tol": back(o_tol), "lse": lse,
           "lse_tol": torch.where(empty, 0.0, es[..., 0] + (Skv + 16) * e32 + 8 * e32 * torch.where(empty, 0.0, lse).abs())}
    if d_o is not None:
        g = torch.where(row_used[:, None, :, None], heads(d_o.detach().cpu().double()), 0.0)
        dp = g @ V.transpose(2, 3)
        delta = (g * o).sum(dim=3, keepdim=True)
        slope = (1 - t * t if cap else torch.ones_like(x)) * scale
        ds = p * (dp - delta) * slope
        # dP, delta (from O as it was stored) and the tanh's derivative, each with its own error
        dp_size = g.abs() @ V.abs().transpose(2, 3)
        dp_tol = (D + 8) * e32 * dp_size
        delta_tol = (g.abs() * (o_tol + (D + 8) * e32 * o.abs())).sum(dim=3, keepdim=True)
        slope_tol = (4 * es / cap if cap else 0.0) * scale + 16 * e32 * scale
        ds_tol = p * (dp_tol + delta_tol) * slope + p * (dp - delta).abs() * (slope * ep + slope_tol) + unit * ds.abs()
        n_q, n_k = (Sq * G + 16) * e32, (Skv + 16) * e32
        dq = ds @ K
        dq_tol = (ds_tol + n_k * ds.abs()) @ K.abs() + unit * dq.abs()

        def shared(a):
            return a.view(B, KH, G, Skv, a.shape[-1]).sum(dim=2)

        dst, pt = ds.transpose(2, 3), p.transpose(2, 3)
        dk, dv = shared(dst @ Q), shared(pt @ g)
        dk_tol = shared((ds_tol + n_q * ds.abs()).transpose(2, 3) @ Q.abs()) + unit * dk.abs()
        dv_tol = shared((pt * (unit + n_q) + (p * ep).transpose(2, 3)) @ g.abs()) + unit * dv.abs()
        out.update(dq=back(dq), dq_tol=back(dq_tol), dk=back(dk), dk_tol=back(dk_tol), dv=back(dv), dv_tol=back(dv_tol))
    return out


def check(got, want, name, what=""):
    """`got` within the bound of want[name] everywhere, infinities where they belong."""
    got, ref, tol = got.detach().cpu().double(), want[name], want[name + "_tol"]
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    whole = torch.isfinite(ref)
    assert torch.equal(got[~whole], ref[~whole]), name + ": infinities"
    off = (got - ref).abs()
    # a NaN is off by nothing that compares
    bad = whole & ~(off <= tol + 1e-30)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%s%s: %d of %d values out of bounds, first at %s: %r, wanted %r within %r"
                             % (what, name, int(bad.sum()), bad.numel(), at, got[tuple(at)].item(), ref[tuple(at)].item(), tol[tuple(at)].item()))
