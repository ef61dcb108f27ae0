"""The transformer-layer operators in 64 bits, and how far a right kernel's outputs may be from them.

A rounding to bf16 is off by at most HALF = finfo(bfloat16).eps / 2 = 2^-8 of the value; an fp32 sum of n products by at most n 2^-24 of
the sum of their magnitudes (its exponentials and divisions by a few units of 2^-24 each).  The bounds below carry these through the
formulas element by element; nothing in them was fitted to an output."""
import math

import torch

HALF = torch.finfo(torch.bfloat16).eps / 2
F32 = 2.0 ** -24
TINY = 2.0 ** -126  # fp32 and bf16 hold nothing smaller with full precision: exponentials, weights and products below it become 0


def rotary(x, coords, sections, base, interleaved, inverse=False):
    """(reference, bound without the output's own rounding): pairs as complex numbers."""
    y = x.double().cpu()
    half = sum(sections)
    c = coords.cpu()
    angle = torch.cat([c[..., a, None].double() * torch.exp(-torch.arange(n, dtype=torch.float64) / max(n, 1) * math.log(base))
                       for a, n in enumerate(sections)], -1)[..., None, :]
    turn = torch.polar(torch.ones((), dtype=torch.float64), -angle if inverse else angle)
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(y[..., i].contiguous(), y[..., j].contiguous()) * turn
    out, err = y.clone(), torch.zeros_like(y)
    out[..., i], out[..., j] = z.real, z.imag
    # remainder of the angle rounded to fp32 (<= 2^-24 pi / 4), two Taylor sums and two products: 8 units of 2^-24 of both channels
    # ... and the angle itself, in 64 bits on both sides: a frequency here is exp of a product of up to 9.3 in magnitude (9.3 + 2 units of
    # 2^-53), the kernel's a power, a division by 2 pi and a product with a rounded 2 pi (5 units): 17 units of 2^-53 of the angle
    e = (8 * F32 + 17 * 2.0 ** -53 * angle.abs()) * (y[..., i].abs() + y[..., j].abs())
    err[..., i] = err[..., j] = e
    return out, err


def rounded(ref, err, dtype):
    """The bound of an output stored in `dtype`."""
    return err + torch.finfo(dtype).eps / 2 * (ref.abs() + err) + TINY


def spans(offset, rows, batch, length):
    if offset is None:
        return [(b * length, length) for b in range(batch)]
    ends = offset.tolist()
    return [(lo, max(hi - lo, 0)) for lo, hi in zip([0] + ends[:-1], ends)]


def attention(q, k, v, mask, q_spans, k_spans, scale, dout=None):
    """q (T, H, D), k, v (T', Hkv, D) as flat rows, mask (T') bool or None.  [(reference, bound)] for out, lse (and dq, dk, dv)."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    (_, H, D), hkv = q.shape, k.shape[1]
    group = H // hkv
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    eo, el, eq, ek, ev = torch.zeros_like(q), torch.zeros_like(lse), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    g = dout.double().cpu() if dout is not None else None
    for (q0, qn), (k0, kn) in zip(q_spans, k_spans):
        keys = torch.arange(k0, k0 + kn)
        if mask is not None:
            keys = keys[~mask.cpu()[k0:k0 + kn]]
        if qn == 0 or len(keys) == 0:
            continue
        for h in range(H):
            Q, K, V = q[q0:q0 + qn, h], k[keys, h // group], v[keys, h // group]
            s = Q @ K.T * scale
            # fp32 scores: D products and sums, the scaled difference and its exponential
            es = scale * (D + 4) * F32 * (Q.abs() @ K.abs().T) + 16 * F32 * (1 + s.abs().amax(-1, keepdim=True))
            big = s.amax(-1, keepdim=True)
            w = torch.exp(s - big)
            l = w.sum(-1, keepdim=True)
            p = w / l
            top = (p * es).sum(-1, keepdim=True)          # relative error of the sum of exponentials
            ep = p * (es + top + (len(keys) + 8) * F32) + TINY  # absolute error of a weight
            out[q0:q0 + qn, h] = o = p @ V
            lse[q0:q0 + qn, h] = (big + l.log()).squeeze(-1)
            # a weight meets V after its rounding to bf16; n + 2 roundings of the fp32 sum
            eo[q0:q0 + qn, h] = eoo = (ep + HALF * p + (len(keys) + 8) * F32 * p) @ V.abs()
            el[q0:q0 + qn, h] = (top + (len(keys) + 32) * F32 * (1 + big.abs() + l.log())).squeeze(-1)
            if g is None:
                continue
            G = g[q0:q0 + qn, h]
            dp = G @ V.T
            delta = (G * o).sum(-1, keepdim=True)
            edp = (D + 4) * F32 * (G.abs() @ V.abs().T)
            # delta from the output as it was stored, at worst (kept in fp32 it is closer)
            ed = (G.abs() * (eoo + HALF * (o.abs() + eoo))).sum(-1, keepdim=True) + (D + 4) * F32 * (G.abs() * o.abs()).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            # weights recomputed from lse: its error once more
            ep2 = ep + p * el[q0:q0 + qn, h, None]
            eds = ep2 * ((dp - delta).abs() + edp + ed) + p * (edp + ed)
            eds = eds + HALF * (ds.abs() + eds) + TINY
            dq[q0:q0 + qn, h] = scale * ds @ K
            eq[q0:q0 + qn, h] = scale * ((eds + (len(keys) + 8) * F32 * ds.abs()) @ K.abs())
            n = qn * group
            dk[keys, h // group] += scale * ds.T @ Q
            ek[keys, h // group] += scale * ((eds + (n + 8) * F32 * ds.abs()).T @ Q.abs())
            dv[keys, h // group] += p.T @ G
            ev[keys, h // group] += (ep2 + HALF * (p + ep2) + (n + 8) * F32 * p).T @ G.abs()
    got = [(out, rounded(out, eo, torch.bfloat16)), (lse, el + 4 * F32 * lse.abs().nan_to_num(posinf=0.0))]
    if g is not None:
        got += [(t, rounded(t, e, torch.bfloat16)) for t, e in ((dq, eq), (dk, ek), (dv, ev))]
    return got


def _act(a, kind):
    """act, act', and the largest |act'| and |act''|."""
    if kind == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s)), 1.1, 0.5
    if kind == "gelu":
        c = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        return a * c, c + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi), 1.13, 0.8
    return a.clamp_min(0), (a > 0).double(), 1.0, 0.0


def ffn(x, wg, wu, wd, bg, bu, bd, kind, dy=None):
    """[(reference, bound)] for y (and dx, dwg, dwu, dwd, dbg, dbu, dbd)."""
    x, wg, wu, wd = (t.double().cpu() for t in (x, wg, wu, wd))
    R, E = x.shape
    F = wg.shape[0]
    zero = torch.zeros((), dtype=torch.float64)
    bg, bu, bd = (b.double().cpu() if b is not None else zero for b in (bg, bu, bd))
    a, u = x @ wg.T + bg, x @ wu.T + bu
    ea = (E + 4) * F32 * (x.abs() @ wg.abs().T + bg.abs())
    eu = (E + 4) * F32 * (x.abs() @ wu.abs().T + bu.abs())
    s, ds, m1, m2 = _act(a, kind)
    h = s * u
    # the activation to 16 units of fp32 (an exponential or error function, a division, a product)
    es = m1 * ea + 16 * F32 * (s.abs() + a.abs())
    eh = es * u.abs() + s.abs() * eu + es * eu
    eh = eh + HALF * (h.abs() + eh)
    y = h @ wd.T + bd
    got = [(y, rounded(y, eh @ wd.abs().T + (F + 4) * F32 * (h.abs() @ wd.abs().T + bd.abs()), torch.bfloat16))]
    if dy is None:
        return got
    g = dy.double().cpu()
    dh = g @ wd
    edh = (E + 4) * F32 * (g.abs() @ wd.abs())
    da, du = dh * u * ds, dh * s
    # a and u as bf16 at worst (kept in fp32 they are closer)
    sa, su = ea + HALF * (a.abs() + ea), eu + HALF * (u.abs() + eu)
    eds = m2 * sa + 16 * F32 * (1 + a.abs())
    if kind == "relu":
        eds = eds + (a.abs() <= ea).double()  # a sum that close to zero may be on either side of it
    es2 = m1 * sa + 16 * F32 * (s.abs() + a.abs())
    eda = edh * (u.abs() + su) * (ds.abs() + eds) + dh.abs() * (su * (ds.abs() + eds) + u.abs() * eds)
    edu = edh * (s.abs() + es2) + dh.abs() * es2
    eda, edu = eda + HALF * (da.abs() + eda), edu + HALF * (du.abs() + edu)
    both = da.abs() @ wg.abs() + du.abs() @ wu.abs()
    dx = da @ wg + du @ wu
    res = [(dx, eda @ wg.abs() + edu @ wu.abs() + (2 * F + 4) * F32 * both)]
    for d, e in ((da, eda), (du, edu)):
        res.append((d.T @ x, e.T @ x.abs() + (R + 4) * F32 * (d.abs().T @ x.abs())))
    res.append((g.T @ h, g.abs().T @ eh + (R + 4) * F32 * (g.abs().T @ h.abs())))
    res += [(d.sum(0), e.sum(0) + (R + 4) * F32 * d.abs().sum(0)) for d, e in ((da, eda), (du, edu), (g, torch.zeros_like(g)))]
    return got + [(t, rounded(t, e, torch.bfloat16)) for t, e in res]


def check(got, ref, bound, what):
    got, ref, bound = got.detach().double().cpu(), ref.detach(), bound.detach()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same = got == ref  # infinities
    bad = ~(same | ((got - ref).abs() <= bound))
    assert not bad.any(), "%s: %d of %d values off, the worst by %.3g of its bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / bound.clamp_min(1e-300))[bad].nan_to_num(nan=math.inf).max()))
