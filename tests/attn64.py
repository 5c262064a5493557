"""Attention with a causal window and sinks in 64 bits, its gradients, and how far a
kernel's results may be from them.

The bounds count roundings.  With u = eps / 2 of the storage type (bf16 2^-8, fp32
2^-24), e = 2^-24 and sums of N terms in fp32 off by at most N e times the sum of
the terms' magnitudes:

  a logit in log2 units   x = c q.k:  off by  (d + 4) e c sum |q||k|  (products and
                          their sum, the factor, the shift)  =: dx, so that
                          p = 2^(x - lse) is off by  r = 2 dx + 8 e  relative, lse's
                          own error being at most the largest dx of its row
  o = sum p v             each p also rounded to the storage type (u), the quotient
                          and the result rounded:  (r + u + N e) sum p|v| + (u + 2 e)|o|
  D = sum do o            (d e + u) sum |do||o| + sum |do| (error of o)
  ds = p (do.v - D)       r |ds| + p (d e sum |do||v| + error of D), rounded: + u |ds|
  dq, dk = scale sum ds k   sums of the above's magnitudes, + N e, rounded: u
  dv = sum p do           (r + u + N e) sum p|do|, rounded: u

Below fp32's normal range a p or a result may be 0 instead: every p is off by up to
f = 2^-126 besides, which adds f sum |v| to o, f (|do.v| + |D|) to a ds, f sum |do| to
dv, and f to each result.
"""
import torch

E = 2.0 ** -24
F = 2.0 ** -126


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def visible(i, j, window, sinks):
    """Whether query positions i see key positions j (window None: every earlier key)."""
    i, j = i[:, None], j[None]
    see = j <= i
    if window is not None:
        see &= (j > i - window) | (j < sinks)
    return see


def attend(q, k, v, see, scale, u, dout=None, qerr=None):
    """One KV head: q [rows, G, d], k, v [keys, d], see [rows, keys]; rows that see
    nothing are 0.  Returns (o, bound) and with dout ((o, dq, dk, dv), bounds); inputs
    of any type, computed in 64 bits.  qerr: how far the kernel's queries may be from q."""
    q, k, v = q.double(), k.double(), v.double()
    G, d = q.shape[1:]
    N = see.shape[1] + G * see.shape[0]
    sees = see[None]
    qh = q.transpose(0, 1)                                        # [G, rows, d]
    x = torch.where(sees, qh @ k.T * scale, torch.full((), -torch.inf, dtype=torch.float64))
    some = see.any(1)[None, :, None]
    p = torch.where(some, torch.softmax(x, -1).nan_to_num(0.0), torch.zeros((), dtype=torch.float64))
    dx = (d + 4) * E * scale * 1.4427 * (qh.abs() @ k.abs().T)
    if qerr is not None:
        dx = dx + scale * 1.4427 * (qerr.double().transpose(0, 1) @ k.abs().T)
    dx = torch.where(sees, dx, torch.zeros((), dtype=torch.float64)).amax(-1, keepdim=True)
    r = 2 * dx + 8 * E
    o = p @ v
    f = F * sees.double()
    bo = (r + u + N * E) * (p @ v.abs()) + (u + 2 * E) * o.abs() + f @ v.abs() + F
    if dout is None:
        return o.transpose(0, 1), bo.transpose(0, 1)
    do = dout.double().transpose(0, 1)
    dp = do @ v.T
    D = (do * o).sum(-1, keepdim=True)
    bD = (d * E + u) * (do * o).abs().sum(-1, keepdim=True) + (do.abs() * bo).sum(-1, keepdim=True)
    ds = p * (dp - D)
    bds = (r + u) * ds.abs() + p * (d * E * (do.abs() @ v.abs().T) + bD) + f * (dp.abs() + D.abs())
    dq, dk, dv = ds @ k * scale, (ds.transpose(1, 2) @ qh).sum(0) * scale, (p.transpose(1, 2) @ do).sum(0)
    bq = scale * ((bds + N * E * ds.abs()) @ k.abs()) + (u + 2 * E) * dq.abs() + F
    bk = scale * ((bds + N * E * ds.abs()).transpose(1, 2) @ qh.abs()).sum(0) + (u + 2 * E) * dk.abs() + F
    bv = ((r + u + N * E) * p + f).transpose(1, 2) @ do.abs()
    bv = bv.sum(0) + (u + 2 * E) * dv.abs() + F
    t = lambda z: z.transpose(0, 1)  # noqa: E731
    return (t(o), t(dq), dk, dv), (t(bo), t(bq), bk, bv)


def norm_rotate(x, gain, eps, cos, sin, u):
    """QKNorm (gain None: none) and rotation of x [rows, H, d] with cos, sin [rows, d]
    in 64 bits: (normalised, rotated, error of the rotated in fp32 and one rounding u).
    The norm: d e / 2 from the sum of squares, 6 e from root, division, gain, scale; the
    rotation 3 e of both products' magnitudes."""
    x = x.double()
    d = x.shape[-1]
    if gain is not None:
        x = x / x.square().mean(-1, keepdim=True).clamp_min(eps).sqrt() * gain.double()[:, None]
    if cos is None:
        return x, x, (d / 2 + 6 + u / E) * E * x.abs()
    h = d // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    other = torch.cat((-x[..., h:], x[..., :h]), -1)
    y = x * c + other * s
    return x, y, (d / 2 + 9) * E * (x.abs() * c.abs() + other.abs() * s.abs()) + u * y.abs()


def sliding(q, k, v, window, sinks, scale, lens, u, dout=None):
    """A batch: q [B, n, Hq, d], k, v [B, n, Hkv, d] on the CPU.  Returns the results
    (out or (out, dq, dk, dv)) and their bounds, 0 in padding."""
    B, n, Hq, d = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    shapes = [q.shape] if dout is None else [q.shape, q.shape, k.shape, k.shape]
    res = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    bnd = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    for b in range(B):
        m = n if lens is None else int(lens[b])
        if m <= 0:
            continue
        i = torch.arange(m)
        see = visible(i, i, window, sinks)
        for h in range(Hkv):
            hs = slice(h * G, h * G + G)
            got, bound = attend(q[b, :m, hs], k[b, :m, h], v[b, :m, h], see, scale, u,
                                None if dout is None else dout[b, :m, hs])
            got, bound = ((got,), (bound,)) if dout is None else (got, bound)
            for to, frm in ((res, got), (bnd, bound)):
                for x, y in zip(to[:2], frm[:2]):
                    x[b, :m, hs] = y
                for x, y in zip(to[2:], frm[2:]):
                    x[b, :m, h] = y
    return (res[0], bnd[0]) if dout is None else (res, bnd)


def assert_within(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    over = err - bound
    worst = int(over.argmax())
    assert bool((err <= bound).all()), (
        f"{what}: {int((~(err <= bound)).sum())} of {err.numel()} values off by more than their bound; worst "
        f"{err.flatten()[worst]:.3g} against {bound.flatten()[worst]:.3g} at value {want.flatten()[worst]:.3g}")
