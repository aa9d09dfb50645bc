"""Cases, plain forms and exact values of the kernel products over sequences (f3m_amd.sequence): attention with a
sliding window and a few first tokens that stay visible, and linear attention with a decay for each head.

Layouts: q (B, Nq, Hq, D), k and v (B, Nk, Hkv, D); linear attention q, k (B, N, H, Dk), v (B, N, H, Dv), state
(B, H, Dk, Dv) in fp32.  The plain forms write the whole matrix of products in 32 bits."""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NBYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def attn(name, dtype, train, B, Nq, Nk, Hq, Hkv, D, window, sinks, ragged):
    return dict(name=name, op="attn", dtype=dtype, train=train, B=B, Nq=Nq, Nk=Nk, Hq=Hq, Hkv=Hkv, D=D, window=window,
                sinks=sinks, ragged=ragged)


def linear(name, dtype, mode, B, N, H, Dk, Dv, ragged):
    return dict(name=name, op="linear", dtype=dtype, mode=mode, B=B, N=N, H=H, Dk=Dk, Dv=Dv, ragged=ragged)


def listed():
    return [
        # one token of one sequence in a small model, the window inside a cache that just left it: latency
        attn("attn token", "bf16", False, 1, 1, 257, 8, 8, 64, 128, 4, False),
        # a serving step: one token for each of many sequences whose caches are filled to different lengths, long window
        attn("attn tokens long", "bf16", False, 32, 1, 32768, 32, 8, 128, 8192, 4, True),
        # a prompt that arrives in chunks: 512 new tokens each over caches of different lengths, no window
        attn("attn chunk", "fp16", False, 4, 512, 8192, 16, 4, 128, 0, 0, True),
        # a whole prompt of one user with a window and sinks
        attn("attn prompt", "bf16", False, 1, 8192, 8192, 32, 8, 128, 1024, 16, False),
        # a training step's layer with a window and sinks, grouped heads
        attn("attn train window", "bf16", True, 2, 4096, 4096, 16, 4, 128, 1024, 4, False),
        # a training step's layer that sees the whole context, small heads, one k/v head for each
        attn("attn train whole", "bf16", True, 1, 4096, 4096, 16, 16, 64, 0, 0, False),
        # fine-tuning in 32 bits on a padded batch of odd lengths with an odd head size
        attn("attn train padded", "fp32", True, 3, 777, 777, 6, 2, 80, 100, 3, True),
        # one token of one sequence, 32-bit model
        linear("linear token", "fp32", "step", 1, 1, 4, 64, 64, False),
        # a serving step: one token for each of many sequences, the states are most of what is moved
        linear("linear tokens many", "bf16", "step", 256, 1, 16, 128, 128, False),
        # a whole prompt of one user, the state goes on to the single tokens
        linear("linear prompt", "bf16", "prompt", 1, 8192, 32, 128, 128, False),
        # a training step's layer
        linear("linear train", "bf16", "train", 4, 2048, 16, 128, 128, False),
        # training through time on a padded batch of odd lengths: the state comes from the piece before and its gradient goes back
        linear("linear train padded", "fp16", "train", 3, 1001, 5, 64, 96, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.55:
        D, Hkv = rng.choice([32, 64, 80, 96, 128]), rng.choice([1, 2, 3, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 5, 8])
        window, sinks = rng.choice([0, _log_int(rng, 16, 8192)]), rng.choice([0, rng.randint(1, 64)])
        kind, ragged = rng.choice(["token", "chunk", "prompt", "train"]), rng.random() < 0.5
        if kind == "token":      # at most the cache of the longest listed one
            Nq, Nk = rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 16, 32768)
            B = _log_int(rng, 1, max(1, min(64, (1 << 30) // (Nk * Hkv * D * 2))))
        elif kind == "chunk":
            Nq = _log_int(rng, 8, 1024)
            Nk = Nq + _log_int(rng, 16, 8192)
            B = _log_int(rng, 1, max(1, min(8, (1 << 29) // (Nq * Nk * Hq))))
        else:
            Nq = Nk = _log_int(rng, 40, 6000)
            B = _log_int(rng, 1, max(1, min(8, (1 << (29 if kind == "train" else 30)) // (Nq * Nk * Hq))))
            if kind == "train":  # no more than the listed training steps
                Hq, Hkv = (Hq, Hkv) if Hq <= 16 else (Hkv, Hkv)
                if dtype == "fp32":
                    Nq = Nk = min(Nq, 2048)
        c = attn("", dtype, kind == "train", B, Nq, Nk, Hq, Hkv, D, window, sinks, ragged)
    else:
        Dk, Dv, H = rng.choice([32, 64, 96, 128]), rng.choice([32, 64, 80, 128]), rng.choice([1, 2, 5, 8, 16])
        mode, ragged = rng.choice(["step", "prompt", "train"]), rng.random() < 0.5
        if mode == "step":
            c = linear("", dtype, mode, _log_int(rng, 1, 256), 1, H, Dk, Dv, False)
        else:
            N = _log_int(rng, 20, 8192 if mode == "prompt" else 4096)
            B = _log_int(rng, 1, max(1, min(8, (1 << 28) // (N * N * H))))
            c = linear("", dtype, mode, B, N, H, Dk, Dv, ragged)
    del c["name"]
    return c


def _lengths(g, B, lo, hi):
    n = torch.randint(lo, hi + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = hi
    return n


def prepare(case, seed):
    c, t = case, TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=t, by=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(by)

    s = {"case": c}
    if c["op"] == "attn":
        s["q"] = randn(c["B"], c["Nq"], c["Hq"], c["D"], by=1.5)
        s["k"] = randn(c["B"], c["Nk"], c["Hkv"], c["D"])
        s["v"] = randn(c["B"], c["Nk"], c["Hkv"], c["D"])
        s["q_lens"] = s["kv_lens"] = None
        if c["ragged"]:
            s["kv_lens"] = _lengths(g, c["B"], max(1, c["Nk"] // 4 if c["Nq"] != c["Nk"] else 1), c["Nk"])
            if c["Nq"] == c["Nk"]:             # a padded batch: as many queries as keys in each sequence
                s["q_lens"] = s["kv_lens"]
        if c["train"]:
            s["dout"] = randn(c["B"], c["Nq"], c["Hq"], c["D"])
            for n in "qkv":
                s[n].requires_grad_()
        return s
    H = c["H"]
    # the decays of a layer's heads: memories from two tokens to about two thousand
    s["log_decay"] = -torch.exp2(torch.linspace(-1.0, -11.0, H, device="cuda")) if H > 1 else torch.full((1,), -0.01, device="cuda")
    if c["mode"] == "step":
        s["q"], s["k"] = randn(c["B"], H, c["Dk"]), randn(c["B"], H, c["Dk"], by=c["Dk"] ** -0.5)
        s["v"] = randn(c["B"], H, c["Dv"])
        s["state"] = randn(c["B"], H, c["Dk"], c["Dv"], dtype=torch.float32)
        return s
    s["q"], s["k"] = randn(c["B"], c["N"], H, c["Dk"]), randn(c["B"], c["N"], H, c["Dk"], by=c["Dk"] ** -0.5)
    s["v"] = randn(c["B"], c["N"], H, c["Dv"])
    s["lens"] = _lengths(g, c["B"], 1, c["N"]) if c["ragged"] else None
    s["state0"] = randn(c["B"], H, c["Dk"], c["Dv"], dtype=torch.float32) if c["ragged"] else None
    if c["mode"] == "train":
        s["dout"] = randn(c["B"], c["N"], H, c["Dv"])
        s["dstate"] = randn(c["B"], H, c["Dk"], c["Dv"], dtype=torch.float32) if c["ragged"] else None
        for n in ("q", "k", "v") + (("state0",) if c["ragged"] else ()):
            s[n].requires_grad_()
    return s


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        if state["case"]["op"] == "attn":
            return _plain_attention(state)
        return _plain_step(state) if state["case"]["mode"] == "step" else _plain_linear(state)


# ---- the framework's calls ---------------------------------------------------------------------------

def _own(s):
    from f3m_amd import sequence
    c = s["case"]
    if c["op"] == "attn":
        out = sequence.window_attention(s["q"], s["k"], s["v"], window=c["window"] or None, sinks=c["sinks"],
                                        q_lens=s["q_lens"], kv_lens=s["kv_lens"])
        if not c["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    if c["mode"] == "step":
        out = sequence.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return out, s["state"]
    out, last = sequence.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state0"], lens=s["lens"])
    if c["mode"] == "prompt":
        return out, last
    if s["state0"] is None:
        return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return (out.detach(), last.detach()) + torch.autograd.grad((out, last), (s["q"], s["k"], s["v"], s["state0"]),
                                                               (s["dout"], s["dstate"]))


# ---- plain forms --------------------------------------------------------------------------------------

def _rows(x, Hkv):
    """(B, N, Hkv G, D) -> (B, Hkv, G N, D) in 32 bits: the rows that share a k/v head."""
    B, N, H, D = x.shape
    return x.float().view(B, N, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, H // Hkv * N, D)


def _unrows(x, N, dtype):
    B, Hkv, R, D = x.shape
    return x.view(B, Hkv, R // N, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hkv * (R // N), D).to(dtype)


def _plain_attention(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    B, Nq, Nk, Hkv, G, D = c["B"], c["Nq"], c["Nk"], c["Hkv"], c["Hq"] // c["Hkv"], c["D"]
    full = lambda n: torch.full((B,), n, device="cuda", dtype=torch.int32)  # noqa: E731
    q_len, kv_len = (full(n) if x is None else x for n, x in ((Nq, s["q_lens"]), (Nk, s["kv_lens"])))
    i, j = torch.arange(Nq, device="cuda"), torch.arange(Nk, device="cuda")
    p = ((kv_len - q_len)[:, None] + i)[:, :, None]
    see = (j <= p) & (i < q_len[:, None])[:, :, None]
    if c["window"]:
        see = see & ((j > p - c["window"]) | (j < c["sinks"]))
    see = see[:, None, None].expand(B, 1, G, Nq, Nk).reshape(B, 1, G * Nq, Nk)
    scale = D ** -0.5
    qr, kr, vr = _rows(q, Hkv), _rows(k, Hkv), _rows(v, Hkv)
    w = torch.matmul(qr, kr.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(~see, float("-inf"))
    top = w.amax(3, keepdim=True).clamp_(min=-3e38)
    w = w.sub_(top).exp_()
    total = w.sum(3, keepdim=True)
    w = w.div_(total.clamp(min=1e-38))
    out = torch.matmul(w, vr)
    if not c["train"]:
        return _unrows(out, Nq, q.dtype)
    do = _rows(s["dout"], Hkv)
    dv = torch.matmul(w.transpose(2, 3).contiguous(), do)
    dw = torch.matmul(do, vr.transpose(2, 3).contiguous())
    dw = dw.sub_((do * out).sum(3, keepdim=True)).mul_(w).mul_(scale)
    dq = torch.matmul(dw, kr)
    dk = torch.matmul(dw.transpose(2, 3).contiguous(), qr)
    return _unrows(out, Nq, q.dtype), _unrows(dq, Nq, q.dtype), _unrows(dk, Nk, k.dtype), _unrows(dv, Nk, v.dtype)


def _plain_step(s):
    q, k, v, S = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    S.mul_(s["log_decay"].double().exp().float()[None, :, None, None]).add_(k[..., None] * v[..., None, :])
    out = (q[..., None] * S).sum(2) * q.shape[-1] ** -0.5
    return out.to(s["v"].dtype), S


def _plain_linear(s):
    c, N = s["case"], s["case"]["N"]
    scale, g = c["Dk"] ** -0.5, s["log_decay"].double()
    q, k, v = (s[n].float().transpose(1, 2).contiguous() for n in "qkv")          # (B, H, N, D)
    t = torch.arange(N, device="cuda")
    n = torch.full((c["B"],), N, device="cuda") if s["lens"] is None else s["lens"].long()
    valid = (t < n[:, None])[:, None, :, None]                                      # (B, 1, N, 1)
    q, k, v = q * valid, k * valid, v * valid
    powers = torch.exp(g[:, None] * torch.arange(N + 1, device="cuda")).float()   # (H, N + 1): decay to the power of a distance
    d = t[:, None] - t
    w = powers[:, d.clamp(min=0)] * (d >= 0) * scale                                # (H, N, N)
    S0 = torch.zeros(c["B"], c["H"], c["Dk"], c["Dv"], device="cuda") if s["state0"] is None else s["state0"]
    from0 = powers[:, 1:, None]                                                      # decay from the state before to token t
    left = (n[:, None] - 1 - t).clamp(min=0)                                         # tokens from t to the last one
    to_end = torch.gather(powers[None].expand(c["B"], -1, -1), 2, left[:, None].expand(-1, c["H"], -1))[..., None]
    over = torch.gather(powers[None].expand(c["B"], -1, -1), 2, n[:, None, None].expand(-1, c["H"], 1))[..., None]
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(w)
    out = torch.matmul(a, v) + torch.matmul(q, S0) * from0 * scale
    back = lambda x, like: (x * valid).transpose(1, 2).to(like.dtype).contiguous()  # noqa: E731
    res = [back(out, s["v"])]
    if c["mode"] == "prompt" or s["state0"] is not None:
        res.append(torch.matmul((k * to_end).transpose(2, 3).contiguous(), v) + S0 * over)
    if c["mode"] == "prompt":
        return tuple(res)
    do = s["dout"].float().transpose(1, 2).contiguous() * valid
    dS = torch.zeros_like(S0) if s["dstate"] is None else s["dstate"]
    dv = torch.matmul(a.transpose(2, 3).contiguous(), do) + torch.matmul(k, dS) * to_end
    da = torch.matmul(do, v.transpose(2, 3).contiguous()).mul_(w)
    dq = torch.matmul(da, k) + torch.matmul(do, S0.transpose(2, 3).contiguous()) * from0 * scale
    dk = torch.matmul(da.transpose(2, 3).contiguous(), q) + torch.matmul(v, dS.transpose(2, 3).contiguous()) * to_end
    res += [back(dq, s["q"]), back(dk, s["k"]), back(dv, s["v"])]
    if s["state0"] is not None:
        res.append(torch.matmul((q * from0).transpose(2, 3).contiguous(), do) * scale + dS * over)
    return tuple(res)


# ---- exact values -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attention(s)
    return _exact_step(s) if case["mode"] == "step" else _exact_linear(s)


def _exact_attention(s):
    """Sequence by sequence and head by head, the visible keys of each row by its definition; gradients by differentiation."""
    c = s["case"]
    G = c["Hq"] // c["Hkv"]
    res = {n: torch.zeros(s[n].shape, device="cuda", dtype=torch.float64) for n in ("q", "k", "v")}
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b in range(c["B"]):
        nk = c["Nk"] if s["kv_lens"] is None else int(s["kv_lens"][b])
        nq = c["Nq"] if s["q_lens"] is None else int(s["q_lens"][b])
        at = torch.arange(nk - nq, nk, device="cuda")[:, None]
        key = torch.arange(nk, device="cuda")[None]
        hide = key > at
        if c["window"]:
            hide |= (at - key >= c["window"]) & (key >= c["sinks"])
        for h in range(c["Hq"]):
            q, k, v = (x[b, :n, i].detach().double().requires_grad_(c["train"])
                       for x, n, i in ((s["q"], nq, h), (s["k"], nk, h // G), (s["v"], nk, h // G)))
            p = torch.softmax((q @ k.t() / c["D"] ** 0.5).masked_fill(hide, float("-inf")), dim=1)
            o = torch.where(hide.all(1, keepdim=True), torch.zeros((), device="cuda", dtype=torch.float64), p @ v)
            out[b, :nq, h] = o.detach()
            if c["train"]:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["dout"][b, :nq, h].double())
                res["q"][b, :nq, h] = dq
                res["k"][b, :nk, h // G] += dk
                res["v"][b, :nk, h // G] += dv
    return (out, res["q"], res["k"], res["v"]) if c["train"] else out


def _exact_step(s):
    S = torch.exp(s["log_decay"].double())[:, None, None] * s["state"].double()
    S = S + torch.einsum("bhi,bhj->bhij", s["k"].double(), s["v"].double())
    return torch.einsum("bhi,bhij->bhj", s["q"].double(), S) / s["q"].shape[-1] ** 0.5, S


def _exact_linear(s):
    """Token by token: the state's recurrence forwards, its adjoint's backwards."""
    c = s["case"]
    B, N, H, Dk, Dv = c["B"], c["N"], c["H"], c["Dk"], c["Dv"]
    lam, root = torch.exp(s["log_decay"].double())[None, :, None, None], Dk ** 0.5
    q, k, v = (s[n].detach().double() for n in "qkv")
    lens = [N] * B if s["lens"] is None else s["lens"].tolist()
    S = torch.zeros(B, H, Dk, Dv, device="cuda", dtype=torch.float64) if s["state0"] is None else s["state0"].detach().double()
    live = torch.tensor([[t < n for n in lens] for t in range(N)], device="cuda")[:, :, None, None, None]
    out, dq = torch.zeros_like(v), torch.zeros_like(q)
    do = s["dout"].double() if c["mode"] == "train" else None
    for t in range(N):
        S = torch.where(live[t], lam * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        m = live[t][..., 0]
        out[:, t] = torch.matmul(q[:, t, :, None, :], S)[:, :, 0] * m / root
        if do is not None:
            dq[:, t] = torch.matmul(S, do[:, t, :, :, None])[..., 0] * m / root
    res = [out] + ([S] if c["mode"] == "prompt" or s["state0"] is not None else [])
    if do is None:
        return tuple(res)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    R = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double()
    for t in reversed(range(N)):
        m = live[t][..., 0]
        here = R + q[:, t, :, :, None] * do[:, t, :, None, :] / root
        dk[:, t] = torch.matmul(here, v[:, t, :, :, None])[..., 0] * m
        dv[:, t] = torch.matmul(k[:, t, :, None, :], here)[:, :, 0] * m
        R = torch.where(live[t], lam * here, R)
    return tuple(res + [dq, dk, dv] + ([R] if s["state0"] is not None else []))


# ---- the work of a pass --------------------------------------------------------------------------------

def work(case):
    """Inputs read once, outputs written once; of a cache, the keys that some row sees.  Lengths at their mean."""
    c, e = case, NBYTES[case["dtype"]]
    if c["op"] == "attn":
        W = c["window"] or c["Nk"]
        square = c["Nq"] == c["Nk"]
        lens = [c["Nk"]] if not c["ragged"] else [c["Nk"] * f for f in ((0.1, 0.3, 0.5, 0.7, 0.9) if square else (0.3, 0.5, 0.7, 0.9))]
        seen = pairs = rows = 0.0
        for n in lens:
            nq = n if square else c["Nq"]
            first = max(0.0, n - nq)                                   # position of the first row
            steps = 64
            pairs += nq / steps * sum(min(p, W) + max(0.0, min(c["sinks"], p - W)) for p in (first + nq * (x + 0.5) / steps for x in range(steps)))
            seen += min(n, min(n, nq + W - 1) + min(c["sinks"], max(0.0, n - nq - W + 1)))
            rows += nq
        pairs, seen, rows = (x / len(lens) * c["B"] for x in (pairs, seen, rows))
        q, kv = rows * c["Hq"] * c["D"] * e, 2 * seen * c["Hkv"] * c["D"] * e
        whole_q, whole_kv = c["B"] * c["Nq"] * c["Hq"] * c["D"] * e, 2 * c["B"] * c["Nk"] * c["Hkv"] * c["D"] * e
        if not c["train"]:
            return {"bytes": q + kv + whole_q, "flops": 4.0 * pairs * c["Hq"] * c["D"]}
        # forward: q, k, v in, out; backward: q, k, v, out, dout in, the gradients out
        return {"bytes": 4 * q + 2 * kv + 2 * whole_q + whole_kv, "flops": 14.0 * pairs * c["Hq"] * c["D"]}
    Dk, Dv, heads = c["Dk"], c["Dv"], c["B"] * c["H"]
    tokens, held = heads * c["N"] * (0.5 if c["ragged"] else 1.0), heads * Dk * Dv * 4
    if c["mode"] == "step":
        return {"bytes": tokens * (2 * Dk + 2 * Dv) * e + 2 * held, "flops": 5.0 * heads * Dk * Dv}
    once = tokens * (2 * Dk + 2 * Dv) * e
    if c["mode"] == "prompt":
        return {"bytes": once + held * (2 if c["ragged"] else 1), "flops": 4.0 * tokens * Dk * Dv}
    return {"bytes": once + tokens * (4 * Dk + 3 * Dv) * e + (4 * held if c["ragged"] else 0), "flops": 12.0 * tokens * Dk * Dv}
