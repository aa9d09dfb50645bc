"""CPU checks of the sequence products at the ends of their ranges (the kernel sources in the CPU emulation)."""
import pytest
import torch

import sequence_reference as ref
from test_emu_sequence import emu_lib, seq  # noqa: F401


SHARED_BY_MANY = [
    # Nk, window, kv_lens: tiles of keys whose rows, times the 16384 query heads of the key head, lie beyond 32 bits
    (131300, None, [5]),                                            # tiles far behind a short sequence
    (160600, 16, None),                                             # tiles far before the window
]


@pytest.mark.parametrize("case", range(len(SHARED_BY_MANY)))
def test_gradients_of_tiles_that_no_row_sees_in_emulation(seq, case):
    Nk, window, kl = SHARED_BY_MANY[case]
    G = 16384
    q, k, v, dout = ref.make_attention(1, 1, Nk, 1, 1, 8, "fp32", 3, "cpu")
    kw = dict(window=window, kv_lens=None if kl is None else torch.tensor(kl))
    many = lambda x: x.expand(1, 1, G, 8)  # noqa: E731
    out, lse = seq.window_attention(many(q), k, v, return_lse=True, **kw)
    dq, dk, dv = seq.window_attention_grad(many(q), k, v, out, lse, many(dout), **kw)
    one = ref.attention(q, k, v, dout, **kw)
    for g in (0, G - 1):
        ref.check((out[:, :, g:g + 1], dq[:, :, g:g + 1]), one, ("out", "dq"))
    # every head alike: G times the gradients of one, a sum of G equal terms in fp32
    want = {n: (G * one[n][0], G * one[n][1] + (G + 32) * ref.W * G * one[n][0].abs()) for n in ("dk", "dv")}
    ref.check((dk, dv), want, ("dk", "dv"))


def halves(B, N, Hq, Hkv, D, seed, device, by_qk, by_v, by_dout):
    q, k, v, dout = ref.make_attention(B, N, N, Hq, Hkv, D, "fp32", seed, device)
    return tuple((by * x).half() for x, by in ((q, by_qk), (k, by_qk), (v, by_v), (dout, by_dout)))


HALF_GRADIENTS = [
    # N, Hq, Hkv, D, window, sizes of q and k, v, dout
    (6, 2, 1, 128, None, 0.5, 2.0, 7500.0),                          # dout under a loss scale: dS beyond 65504
    (150, 2, 2, 64, 40, 0.5, 4.0, 4096.0),
    (200, 2, 1, 64, None, 4.0, 1.0, 1e-3),                           # no loss scale: dS below fp16's normal numbers
    (200, 4, 2, 32, 50, 4.0, 1.0, 1e-4),
]


@pytest.mark.parametrize("case", range(len(HALF_GRADIENTS)))
def test_gradients_in_half_precision_of_any_size_in_emulation(seq, case):
    N, Hq, Hkv, D, window, by_qk, by_v, by_dout = HALF_GRADIENTS[case]
    q, k, v, dout = halves(2, N, Hq, Hkv, D, case, "cpu", by_qk, by_v, by_dout)
    kw = dict(window=window, sinks=1)
    want = ref.attention(q, k, v, dout, tight=("dS",), **kw)
    assert all(float(want[n][0].abs().max()) < 6e4 for n in ("dq", "dk", "dv"))      # fp16 holds the results
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    ref.check(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), want, ("dq", "dk", "dv"))


def test_one_large_difference_in_half_precision_in_emulation(seq):
    """Two keys, v = +-6, dout = 800, 64 wide: dS = 0.5 x 800 x 6 x 64, dq = 384."""
    one = torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cpu")
    pair = torch.cat([one, -one], 1)
    q, k, v, dout = 0 * one, 0.01 * pair, 6 * pair, 800 * one
    kw = dict(q_lens=None, kv_lens=None, scale=0.125)
    want = ref.attention(q, k, v, dout, tight=("dS",), **kw)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    dq, dk, dv = seq.window_attention_grad(q, k, v, out, lse, dout, **kw)
    ref.check((dq, dk, dv), want, ("dq", "dk", "dv"))
    assert 383 < float(dq[0, 0, 0, 0]) < 385


def test_gradients_of_hardly_seen_keys_in_half_precision_in_emulation(seq):
    """Weights of 2^-20 and less under a large dout: dv of such keys is an ordinary number."""
    q, k, v, dout = halves(1, 120, 2, 2, 64, 7, "cpu", 1.0, 1.0, 4000.0)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, :3, :, 0] = 16.0                                            # three keys that are seen 2^23 times as much (scale 1/8: logits of 16)
    want = ref.attention(q, k, v, dout, tight=("dS", "P"))
    assert 2.0 ** -14 < float(want["dv"][0][:, 3:-3].abs().median()) < 0.1
    out, lse = seq.window_attention(q, k, v, return_lse=True)
    dq, _, dv = seq.window_attention_grad(q, k, v, out, lse, dout)  # dk passes fp16's largest number here
    ref.check((dq, dv), want, ("dq", "dv"))


@pytest.mark.parametrize("Nq", [1, 70])
def test_many_small_weights_beside_a_large_one_in_half_precision_in_emulation(seq, Nq):
    """A first key that takes nearly all of each row and holds nothing: out is what the others leave, weights of 2^-20 and less."""
    N = 400
    q, k, v, _ = halves(1, N, 2, 1, 64, 5, "cpu", 1.0, 1.0, 1.0)
    q, v = q[:, -Nq:].clone(), (v.abs() * 500 + 500)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, 0, :, 0], v[:, 0] = 14.0, 0.0                                # a logit of 14
    want = ref.attention(q, k, v, tight=("weights",))
    assert 1e-3 < float(want["out"][0].median()) < 10
    ref.check(seq.window_attention(q, k, v, return_lse=True), want, ("out", "lse"))


def linear_halves(B, N, H, Dk, Dv, seed, device, by_q, by_k, by_v, by_dout):
    q, k, v, dout, s0, ds = ref.make_linear(B, N, H, Dk, Dv, "fp32", seed, device)
    return tuple((by * x).half() for x, by in ((q, by_q), (k, by_k), (v, by_v), (dout, by_dout))) + (s0, ds)


HALF_LINEAR = [
    # N, Dk, Dv, decay, scale, sizes of q, k, v, dout
    (8, 64, 64, -0.1, 1.0, 100.0, 800.0, 0.01, 0.01),               # q.k beyond 65504, out below
    (100, 64, 32, -0.05, None, 200.0, 1600.0, 0.01, 0.1),
    (100, 32, 64, -0.05, 1.0, 0.02, 0.1, 12.0, 800.0),               # dout.v beyond 65504
    (100, 64, 64, -0.05, None, 1e-3, 2e-3, 3000.0, 1.0),             # q.k below fp16's normal numbers
    (100, 64, 64, -0.05, None, 30.0, 200.0, 1e-3, 1e-2),             # dout.v likewise
]


@pytest.mark.parametrize("case", range(len(HALF_LINEAR)))
def test_linear_attention_in_half_precision_of_any_size_in_emulation(seq, case):
    N, Dk, Dv, g, scale, by_q, by_k, by_v, by_dout = HALF_LINEAR[case]
    q, k, v, dout, _, _ = linear_halves(2, N, 1, Dk, Dv, case, "cpu", by_q, by_k, by_v, by_dout)
    g = torch.tensor([g], device="cpu")
    want = ref.linear(q, k, v, g, dout, scale=scale, tight=("weights",))
    assert all(float(want[n][0].abs().max()) < 6e4 for n in ("out", "dq", "dk", "dv"))      # fp16 holds the results
    ref.check(seq.linear_attention(q, k, v, g, scale=scale), want, ("out", "final"))
    ref.check(seq.linear_attention_grad(q, k, v, g, dout, scale=scale)[:3], want, ("dq", "dk", "dv"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,N", [(1, 330), (30, 140)])
def test_a_state_that_only_fades_in_emulation(seq, B, N, dtype):
    """Tokens that add nothing: the state fades by its decay to fp32 accuracy, forwards and backwards, however strong the decay of a chunk; in segments and (many heads) in
    one piece."""
    H = 6
    q, k, v, dout, s0, ds = ref.make_linear(B, N, H, 32, 32, dtype, 1, "cpu")
    g = torch.tensor([0.0, -0.001, -0.01, -0.03, -0.1, -0.2], device="cpu")
    lens = torch.tensor([max(1, N - 4 * b) for b in range(B)], device="cpu")
    kw = dict(initial_state=s0, lens=lens)
    want = ref.linear(q, k, 0 * v, g, 0 * dout, ds, initial=s0, lens=lens)
    out, last = seq.linear_attention(q, k, 0 * v, g, **kw)
    ref.check((out, last), want, ("out", "final"))
    ref.check(seq.linear_attention_grad(q, k, 0 * v, g, 0 * dout, ds, **kw), want, ("dq", "dk", "dv", "dinitial"))


HALF_MOMENTS = [
    # B, N, H, Dk, Dv, decays, sizes of q, k, v, dout
    (1, 200, 1, 64, 64, [-0.02], 1.0, 1.0, 1e-5, 1e-4),
    (1, 150, 2, 32, 96, [-0.5, -8.0], 1.0, 30.0, 1e-3, 1e-3),       # strong decays: the state's gradient holds e^-8 of dout and less
    (20, 70, 10, 32, 32, [-0.01 * 2 ** n for n in range(10)], 1.0, 1.0, 1e-4, 1e-4),       # walked in one piece
]


@pytest.mark.parametrize("case", range(len(HALF_MOMENTS)))
def test_moments_of_small_values_in_half_precision_in_emulation(seq, case):
    """Final moments and the state's gradient are fp32 whatever the size of what they are formed from."""
    B, N, H, Dk, Dv, g, by_q, by_k, by_v, by_dout = HALF_MOMENTS[case]
    q, k, v, dout, _, _ = linear_halves(B, N, H, Dk, Dv, case, "cpu", by_q, by_k, by_v, by_dout)
    g = torch.tensor(g, device="cpu")
    lens = torch.tensor([max(1, N - 3 * b) for b in range(B)], device="cpu")
    want = ref.linear(q, k, v, g, dout, lens=lens, tight=("weights", "moments"))
    out, last = seq.linear_attention(q, k, v, g, lens=lens)
    ref.check((out, last) + seq.linear_attention_grad(q, k, v, g, dout, lens=lens), want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_a_state_of_any_size_in_half_precision_in_emulation(seq):
    """A large state beside small values, and one that fades."""
    for by, g in ((1e30, -0.5), (1e4, -0.02), (1e-6, 0.0)):
        q, k, v, dout, s0, ds = linear_halves(1, 150, 1, 32, 32, 3, "cpu", 0.0 if by > 1e20 else 1e-2, 1.0, 1e-4, 1e-3)
        g = torch.tensor([g], device="cpu")
        want = ref.linear(q, k, v, g, dout, initial=by * s0, tight=("weights", "moments"))
        ref.check(seq.linear_attention(q, k, v, g, initial_state=by * s0), want, ("out", "final"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N", [40, 200])
def test_scales_far_from_one_in_emulation(seq, N, dtype):
    """The gradient of a state passes through whole whatever the scale of the products beside it."""
    q, k, v, dout, s0, ds = ref.make_linear(2, N, 2, 32, 64, dtype, 4, "cpu")
    g = torch.tensor([-0.01, -0.1], device="cpu")
    for scale, by in ((1e-40, 1.0), (-1e-30, 1e10)) + (((1e25, 1e-20),) if dtype != "fp16" else ()):
        dfinal = by * ds
        kw = dict(scale=scale, initial=s0)
        if dtype == "fp16" and by > 1:
            v, k = 1e-3 * v, 1e-3 * k
            dfinal = 1e-4 * dfinal
        want = ref.linear(q, k, v, g, dout, dfinal, **kw)
        ref.check(seq.linear_attention_grad(q, k, v, g, dout, dfinal, scale=scale, initial_state=s0), want, ("dq", "dk", "dv", "dinitial"))


def test_a_step_tells_autograd_that_the_state_changed_in_emulation(seq):
    q, k, v, dout, s0, _ = ref.make_linear(2, 12, 2, 16, 16, "fp32", 2, "cpu")
    g = torch.tensor([-0.1, -0.2], device="cpu")
    q.requires_grad_()
    state = s0.clone()
    out, _ = seq.linear_attention(q, k, v, g, initial_state=state)
    with torch.no_grad():
        version = state._version
        seq.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
        assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, q, dout)
    with torch.inference_mode():                                     # tensors without a version
        inner = s0.clone()
        seq.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, inner)
    assert torch.equal(inner, state)


def test_derivatives_and_traces_that_would_be_dropped_are_refused_in_emulation(seq):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    q, k, v, dout, s0, ds = ref.make_linear(1, 6, 1, 8, 8, "fp32", 2, "cpu")
    g = torch.tensor([-0.1], device="cpu")
    out, lse = seq.window_attention(q, k, v, return_lse=True)
    calls = {
        "window_attention": (seq.window_attention, (q, k, v)),
        "window_attention_grad": (seq.window_attention_grad, (q, k, v, out, lse, dout)),
        "linear_attention": (lambda q, k, v, g, s: seq.linear_attention(q, k, v, g, initial_state=s), (q, k, v, g, s0)),
        "linear_attention_grad": (lambda q, k, v, g, d, e, s: seq.linear_attention_grad(q, k, v, g, d, e, initial_state=s), (q, k, v, g, dout, ds, s0)),
        "linear_attention_step": (seq.linear_attention_step, (q[:, 0], k[:, 0], v[:, 0], g, s0.clone())),
    }
    for name, (f, args) in calls.items():
        for n in range(len(args)):
            with forward_ad.dual_level():
                dual = list(args)
                dual[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
                with pytest.raises(NotImplementedError, match="forward"):
                    f(*dual)
                f(*args)                                              # a level alone is no reason
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda *a: f(*a))(*args)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d", [0, 4, 12, 20, 129, 136])
def test_head_sizes_are_refused_alike_in_all_types_in_emulation(seq, d, dtype):
    from f3m_amd.capi import F3MError
    f = lambda *s: torch.zeros(*s, dtype=ref.TYPES[dtype], device="cpu")  # noqa: E731
    g, x, ok = torch.zeros(2, device="cpu"), f(1, 3, 2, d), f(1, 3, 2, 8)
    lse = torch.zeros(1, 3, 2, device="cpu")
    for call in (lambda: seq.window_attention(x, x, x), lambda: seq.window_attention_grad(x, x, x, x, lse, x),
                 lambda: seq.linear_attention(x, x, ok, g), lambda: seq.linear_attention(ok, ok, x, g), lambda: seq.linear_attention_grad(x, x, x, g, x),
                 lambda: seq.linear_attention_step(x[:, 0], x[:, 0], ok[:, 0], g, torch.zeros(1, 2, d, 8, device="cpu"))):
        with pytest.raises(F3MError) as e:
            call()
        assert e.value.code == 2


def test_lengths_beyond_32_bits_are_taken_into_the_range_in_emulation(seq):
    q, k, v, dout = ref.make_attention(4, 9, 12, 2, 1, 8, "fp32", 2, "cpu")
    far, near = torch.tensor([2 ** 32 + 1, -2 ** 40, 2 ** 31, 5], device="cpu"), torch.tensor([99, -1, 99, 5], device="cpu")
    for kw in ((dict(q_lens=far), dict(q_lens=near)), (dict(kv_lens=far), dict(kv_lens=near))):
        (a, la), (b, lb) = (seq.window_attention(q, k, v, return_lse=True, **x) for x in kw)
        assert torch.equal(a, b) and torch.equal(la, lb)
        for x, y in zip(*(seq.window_attention_grad(q, k, v, a, la, dout, **x) for x in kw)):
            assert torch.equal(x, y)
    q, k, v, dout, s0, ds = ref.make_linear(4, 9, 1, 8, 8, "fp32", 2, "cpu")
    g = torch.tensor([-0.1], device="cpu")
    for x, y in zip(*(seq.linear_attention(q, k, v, g, initial_state=s0, lens=n) + seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=n)
                      for n in (far, near))):
        assert torch.equal(x, y)


def test_windows_and_sinks_of_any_size_in_emulation(seq):
    q, k, v, dout = ref.make_attention(1, 9, 12, 2, 1, 8, "fp32", 2, "cpu")
    want = seq.window_attention(q, k, v)
    for kw in (dict(window=2 ** 63), dict(window=2 ** 64 + 1), dict(window=1, sinks=2 ** 63), dict(window=1, sinks=2 ** 64)):
        assert torch.equal(seq.window_attention(q, k, v, **kw), want)
    for kw in (dict(window=-2 ** 64 + 1), dict(sinks=-2 ** 64 + 1)):
        with pytest.raises(AssertionError):
            seq.window_attention(q, k, v, **kw)


@pytest.mark.parametrize("dtype,B,Nq,Nk,Hq,Hkv,D,window,sinks", [
    ("bf16", 32, 70, 90, 8, 8, 16, 30, 2),                           # 128 rows a workgroup
    ("fp16", 64, 18, 100, 16, 4, 32, 20, 3),                         # 72 rows on one key head
    ("fp32", 64, 40, 70, 8, 4, 8, 9, 1),                              # 80
    ("bf16", 32, 33, 150, 8, 8, 16, 100, 2),                         # 64 rows a workgroup
    ("fp32", 32, 20, 40, 16, 8, 8, None, 0),                         # 40
])
def test_attention_of_many_rows_in_emulation(seq, dtype, B, Nq, Nk, Hq, Hkv, D, window, sinks):
    """Enough rows that wavefronts stand side by side along them."""
    q, k, v, dout = ref.make_attention(B, Nq, Nk, Hq, Hkv, D, dtype, D, "cpu", by=2.0)
    kw = dict(window=window, sinks=sinks, kv_lens=torch.tensor([max(0, Nk - 3 * b) for b in range(B)]))
    want = ref.attention(q, k, v, dout, tight=("dS",) if dtype != "fp32" else (), **kw)      # the second part of dS counts
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, **kw), want, ("out", "lse", "dq", "dk", "dv"))


def test_linear_attention_of_heads_dealt_to_the_xcds_in_emulation(seq):
    B, N, H = 2, 100, 12
    q, k, v, dout, s0, ds = ref.make_linear(B, N, H, 8, 16, "bf16", 5, "cpu")
    g = -0.3 * torch.rand(H, generator=torch.Generator().manual_seed(2))
    lens = torch.tensor([100, 37])
    want = ref.linear(q, k, v, g, dout, ds, initial=s0, lens=lens)
    ref.check(seq.linear_attention(q, k, v, g, initial_state=s0, lens=lens) + seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=lens),
              want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_scales_of_attention_of_any_size_in_emulation(seq):
    """A scale of 0 takes all keys as equal however large the products; a small one is not taken for a larger one; one whose logits fp32 cannot hold is refused."""
    from f3m_amd.capi import F3MError
    q, k, v, dout = ref.make_attention(1, 20, 40, 2, 1, 16, "fp32", 8, "cpu")
    for scale, by in ((0.0, 1e17), (1e-36, 1e17), (-1e-42, 1e18), (1e30, 1e-15)):
        kw = dict(window=9, sinks=2, scale=scale)
        # the library takes the scale as fp32, whose step is 7e-4 of 1e-42
        want = ref.attention(by * q, by * k, v, dout, **dict(kw, scale=float(torch.tensor(scale, dtype=torch.float32))))
        out, lse = seq.window_attention(by * q, by * k, v, return_lse=True, **kw)
        ref.check((out, lse) + seq.window_attention_grad(by * q, by * k, v, out, lse, dout, **kw), want, ("out", "lse", "dq", "dk", "dv"))
    with pytest.raises(F3MError):
        seq.window_attention(q, k, v, scale=3e38)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_a_growing_state_in_emulation(seq, dtype):
    """A log_decay above 0, which the documentation leaves out: the same sums in all types."""
    q, k, v, dout, s0, ds = ref.make_linear(1, 100, 2, 32, 32, dtype, 6, "cpu")
    q, dout = 1e-2 * q, 1e-3 * dout
    g = torch.tensor([0.1, 0.02], device="cpu")
    want = ref.linear(q, k, v, g, dout, 1e-3 * ds, initial=s0)
    assert float(want["out"][0].abs().max()) < 6e4 and float(want["dk"][0].abs().max()) < 6e4
    ref.check(seq.linear_attention(q, k, v, g, initial_state=s0) + seq.linear_attention_grad(q, k, v, g, dout, 1e-3 * ds, initial_state=s0), want,
              ("out", "final", "dq", "dk", "dv", "dinitial"))
