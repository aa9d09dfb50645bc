"""Products over sequences from their definitions in 64 bits, and how far a correct kernel may be from them.

The bounds are sums of worst cases, element by element; u is half a step of the element type (bf16 2^-8, fp16 2^-11, fp32 2^-24)
and w = 2^-24 half a step of the fp32 sums.

* a product of D terms in fp32 is off by at most (D + 2) w times the sum of their magnitudes;
* a weight exp(s) is off by twice the error of s (numerator and row sum) and a few w; weights and their differences
  are rounded once to the element type where they are operands of a product: u of each, in fp16 at least 2^-25
  (its smallest step is 2^-24);
* results are rounded once: u of the result, in fp16 at least 2^-25;
* numbers below 2^-126, the smallest that fp32 and bf16 hold in full, may be taken as 0 by the exponential and by the matrix
  instructions: each weight, and each operand made from one, may be off by 2^-126 whatever its size (a weight exp(-90) = 2^-130 is 0)."""
import torch

W = 2.0 ** -24
FLUSH = 2.0 ** -126
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return 2.0 ** -25 if t == torch.float16 else FLUSH


def visible(nq, nk, window, sinks, device):
    """(nq, nk): row i stands at nk - nq + i."""
    p = torch.arange(nk - nq, nk, device=device)[:, None]
    j = torch.arange(nk, device=device)[None]
    see = j <= p
    if window is not None:
        see &= (p - j < window) | (j < sinks)
    return see


def attention(q, k, v, dout=None, window=None, sinks=0, scale=None, q_lens=None, kv_lens=None, tight=()):
    """-> {name: (value, bound)} for out, lse and, with dout, dq, dk, dv.

    tight names operands whose 16-bit form has no smallest step of its own, because it is taken in units of a power of two: "dS" is a sum of
    two parts (u^2 is lost, and 2^-38 of the largest of a row or key: a part below 2^-24, where the largest is 2^13 or more); "P", the weights for dv, has
    its 1 at 2^15 (half of fp16's smallest step is then 2^-40); "weights", those of the forward pass, has it at 2^7 or more (2^-32)."""
    t, dev = q.dtype, q.device
    u, tiny = half_step(t), least(t)
    B, Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    r = {n: (z(*s), z(*s)) for n, s in (("out", q.shape), ("lse", q.shape[:3]), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape))}
    r["lse"][0].fill_(float("-inf"))
    for b in range(B):
        nq = Nq if q_lens is None else min(max(int(q_lens[b]), 0), Nq)
        nk = Nk if kv_lens is None else min(max(int(kv_lens[b]), 0), Nk)
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, window, sinks, dev)
        some = see.any(1)
        n = see.sum(1, keepdim=True).double()
        for h in range(Hq):
            g = h * Hkv // Hq
            Q, K, V = q[b, :nq, h].detach().double(), k[b, :nk, g].detach().double(), v[b, :nk, g].detach().double()
            s = torch.where(see, scale * (Q @ K.t()), torch.full((), float("-inf"), dtype=torch.float64, device=dev))
            top = s.amax(1, keepdim=True).clamp(min=-1e300)
            e = torch.exp(s - top)
            total = e.sum(1, keepdim=True)
            P = e / total.clamp(min=1e-300)
            O = P @ V
            size = abs(scale) * (torch.where(see, Q.abs() @ K.abs().t(), torch.zeros((), dtype=torch.float64, device=dev))).amax(1, keepdim=True)
            ew = W * (2 * (D + 8) * size + n + 32)                       # of one weight
            seen_v = see.double() @ V.abs()
            bo = (u + ew) * (P @ V.abs()) + ((2.0 ** -32 if "weights" in tight else tiny) + FLUSH) * seen_v + u * O.abs() + tiny
            r["out"][0][b, :nq, h], r["out"][1][b, :nq, h] = O, bo
            lse = (torch.log(total) + top)[:, 0]
            r["lse"][0][b, :nq, h] = torch.where(some, lse, torch.full_like(lse, float("-inf")))
            r["lse"][1][b, :nq, h] = ew[:, 0] + 4 * W * lse.abs().clamp(max=1e30)
            if dout is None:
                continue
            G = dout[b, :nq, h].double()
            dP, delta = G @ V.t(), (G * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            # the weight again, from a stored lse
            ep = ew + W * 8 * lse.abs().clamp(max=1e30)[:, None]
            ep = torch.where(some[:, None], ep, torch.zeros_like(ep))
            bP = u * P + ep * P + ((2.0 ** -40 if "P" in tight else tiny) + FLUSH) * see
            bdelta = (G.abs() * bo).sum(1, keepdim=True) + W * (D + 2) * (G * O).abs().sum(1, keepdim=True)
            tiny_S = 2.0 ** -38 * (dS.abs().amax(1, keepdim=True) + dS.abs().amax(0, keepdim=True)) + FLUSH if "dS" in tight else tiny
            bS = ((2 * u * u if "dS" in tight else u) + ep) * dS.abs() + P * (W * (D + 4) * (G.abs() @ V.abs().t() + (G * O).abs().sum(1, keepdim=True)) + bdelta) + (tiny_S + FLUSH * (dP - delta).abs()) * see
            a = abs(scale)
            rows = W * (nq * Hq // Hkv + 32)
            dq = scale * dS @ K
            r["dq"][0][b, :nq, h] = dq
            r["dq"][1][b, :nq, h] = a * (bS @ K.abs() + W * (n + 32) * (dS.abs() @ K.abs())) + u * dq.abs() + tiny
            r["dk"][0][b, :nk, g] += scale * dS.t() @ Q
            r["dk"][1][b, :nk, g] += a * (bS.t() @ Q.abs() + rows * (dS.abs().t() @ Q.abs()))
            r["dv"][0][b, :nk, g] += P.t() @ G
            r["dv"][1][b, :nk, g] += bP.t() @ G.abs() + rows * (P.t() @ G.abs())
    for n in ("dk", "dv"):
        r[n][1].add_(u * r[n][0].abs() + tiny)
    return r


def _weights(n, g, dev, dtype):
    """Decay to the power of each distance (lower triangle), and the relative error of one that was put together from factors:
    the arguments' and the products' roundings."""
    t = torch.arange(n, device=dev, dtype=torch.float64)
    d = (t[:, None] - t).clamp(min=0)
    low = (t[:, None] >= t).double()
    w = _power(g, d) * low
    return w, W * (2 * g_abs(g) * d + d / 16 + 64)


def g_abs(g):
    return abs(g) if g > -1e30 else 0.0


def _power(g, d):
    if g < -1e30:
        return (d == 0).double()
    return torch.exp(g * d)


def _summed(x, y, z, w, ew, scale, Z, ez, u, tiny, extra, tight=False):
    """out = scale ((w * x y^T) z + x Z) with its bound; x Z: moments that came in, ez: their relative error.  tight: the rows of the
    weights are in units of a power of two that brings the largest of 32 neighbours to 2^13 or more: 2^-38 of a row's largest is lost, not fp16's smallest step."""
    D = x.shape[1]
    a = w * (x @ y.t())
    mag = w * (x.abs() @ y.abs().t())
    s = abs(scale)
    out = scale * (a @ z + x @ Z)
    least_a = FLUSH + 2.0 ** -38 * s * a.abs().amax(1, keepdim=True) if tight else tiny
    b = s * ((u + extra + ew + W * (D + 8)) * mag) @ z.abs() + least_a * (w > 0).double() @ z.abs() + \
        s * (extra + ez + W * (D + 8)) * (x.abs() @ Z.abs())
    return out, b + u * out.abs() + tiny


def linear(q, k, v, log_decay, dout=None, dfinal=None, scale=None, initial=None, lens=None, tight=()):
    """-> {name: (value, bound)} for out, final and, with dout, dq, dk, dv, dinitial.  tight names operands whose 16-bit form has no smallest step
    of its own: "weights", those inside a chunk; "moments", the v of which moments are formed (of two parts, 2^-33 of the largest of a column is lost)."""
    t, dev = q.dtype, q.device
    u, tiny = half_step(t), least(t)
    # moments enter products as two 16-bit parts: 2^-16 of each is a safe bound (bf16 2 x 8 bits, fp16 2 x 11 bits at the largest moment's scale)
    extra = 2.0 ** -16 if t != torch.float32 else 0.0
    B, N, H, Dk = q.shape
    Dv = v.shape[3]
    scale = Dk ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    shapes = (("out", v.shape), ("final", (B, H, Dk, Dv)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("dinitial", (B, H, Dk, Dv)))
    r = {n: (z(*s), z(*s)) for n, s in shapes}
    for b in range(B):
        n = N if lens is None else min(max(int(lens[b]), 0), N)
        for h in range(H):
            g = float(log_decay[h])
            Q, K, V = (x[b, :n, h].detach().double() for x in (q, k, v))
            S0 = z(Dk, Dv) if initial is None else initial[b, h].detach().double()
            G = None if dout is None else dout[b, :n, h].double()
            R0 = z(Dk, Dv) if dfinal is None else dfinal[b, h].double()
            if n == 0:
                r["final"][0][b, h], r["dinitial"][0][b, h] = S0, R0
                r["final"][1][b, h], r["dinitial"][1][b, h] = W * S0.abs(), W * R0.abs()
                continue
            w, ew = _weights(n, g, dev, t)
            one = torch.arange(n, device=dev, dtype=torch.float64)
            from0, left = _power(g, one + 1)[:, None], _power(g, n - 1 - one)[:, None]
            e1 = W * (2 * g_abs(g) * n + n / 16 + 64)
            # moments: each token's term is off by its weight's error and the parts v is split into (2^-22), sums by w each
            part = 2.0 ** -21 + W * 64
            def moments(x, y, f, over, start):
                val = (x * f).t() @ y + over * start
                least_v = FLUSH + 2.0 ** -33 * (f * y.abs()).amax(0, keepdim=True) if "moments" in tight else tiny
                bnd = (part + e1) * ((x * f).abs().t() @ y.abs()) + x.abs().t() @ (least_v * torch.ones_like(y)) + (e1 + W) * over * start.abs()
                return val, bnd + W * val.abs()
            o, bo = _summed(Q, K, V, w, ew, scale, z(Dk, Dv), 0, u, tiny, extra, "weights" in tight)
            # what came in: x Z with a row's own factor
            def came(x, f, Z, s):
                return s * f * (x @ Z), abs(s) * (extra + e1 + W * (Dk + Dv + 8)) * (f * (x.abs() @ Z.abs()))
            c, bc = came(Q, from0, S0, scale)
            r["out"][0][b, :n, h], r["out"][1][b, :n, h] = o + c, bo + bc + u * c.abs()
            over = float(_power(g, torch.tensor(float(n), dtype=torch.float64)))
            r["final"][0][b, h], r["final"][1][b, h] = moments(K, V, left, over, S0)
            if G is None:
                continue
            o, bo = _summed(G, V, K, w, ew, scale, z(Dv, Dk), 0, u, tiny, extra, "weights" in tight)
            c, bc = came(G, from0, S0.t(), scale)
            r["dq"][0][b, :n, h], r["dq"][1][b, :n, h] = o + c, bo + bc + u * c.abs()
            o, bo = _summed(V, G, Q, w.t(), ew.t(), scale, z(Dv, Dk), 0, u, tiny, extra, "weights" in tight)
            c, bc = came(V, left, R0.t(), 1.0)
            r["dk"][0][b, :n, h], r["dk"][1][b, :n, h] = o + c, bo + bc + u * c.abs()
            o, bo = _summed(K, Q, G, w.t(), ew.t(), scale, z(Dk, Dv), 0, u, tiny, extra, "weights" in tight)
            c, bc = came(K, left, R0, 1.0)
            r["dv"][0][b, :n, h], r["dv"][1][b, :n, h] = o + c, bo + bc + u * c.abs()
            d, bd = moments(Q * scale, G, from0, over, R0)
            r["dinitial"][0][b, h], r["dinitial"][1][b, h] = d, bd
    return r


def check(got, want, names):
    """Every element within its bound; infinities equal."""
    for name, x in zip(names, got):
        val, bound = want[name]
        x = x.detach().double()
        assert x.shape == val.shape, (name, x.shape, val.shape)
        inf = torch.isinf(val)
        assert torch.equal(x[inf], val[inf]), name
        off = (x - val).abs()[~inf]
        over = off > bound[~inf]
        if bool(over.any()) or not bool(torch.isfinite(x[~inf]).all()):
            i = int(torch.nan_to_num(off - bound[~inf], nan=1e300).argmax())
            raise AssertionError("%s: %d of %d elements beyond the bound, worst: got %.9g, want %.9g, bound %.3g" % (
                name, int(over.sum()), over.numel(), float(x[~inf][i]), float(val[~inf][i]), float(bound[~inf][i])))


def make_attention(B, Nq, Nk, Hq, Hkv, D, dtype, seed, device, by=1.0):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    f = lambda *s, by=1.0: (by * torch.randn(*s, generator=g)).to(t).to(device)  # noqa: E731
    return f(B, Nq, Hq, D, by=by), f(B, Nk, Hkv, D), f(B, Nk, Hkv, D), f(B, Nq, Hq, D)


def make_linear(B, N, H, Dk, Dv, dtype, seed, device, state=True):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    f = lambda *s, by=1.0: (by * torch.randn(*s, generator=g)).to(t).to(device)  # noqa: E731
    s = lambda: torch.randn(B, H, Dk, Dv, generator=g).to(device) if state else None  # noqa: E731
    return f(B, N, H, Dk), f(B, N, H, Dk, by=Dk ** -0.5), f(B, N, H, Dv), f(B, N, H, Dv), s(), s()
