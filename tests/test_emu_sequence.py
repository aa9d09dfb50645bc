"""CPU checks of the sequence products: the kernel sources in the CPU emulation against the definitions in 64 bits, and the
refusals of the front end and of the C ABI."""
import ctypes as C
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "cpu_emu"))

import sequence_reference as ref  # noqa: E402
from f3m_amd import capi, sequence  # noqa: E402


@pytest.fixture(scope="module")
def emu_lib():
    import build_emu_sequence
    return capi.bind_sequence(C.CDLL(build_emu_sequence.build()))


@pytest.fixture
def seq(emu_lib, monkeypatch):
    """The front end on host tensors, its calls answered by the emulated kernels."""
    class Lib:
        @staticmethod
        def get():
            return emu_lib

    def call(device, name, *args):
        capi.check(emu_lib, getattr(emu_lib, name)(*args, None))

    monkeypatch.setattr(sequence, "_lib", Lib)
    monkeypatch.setattr(sequence, "_call", call)
    monkeypatch.setattr(sequence, "_need_cuda", lambda *t: None)
    return sequence


ATTENTION = [
    # B, Nq, Nk, Hq, Hkv, D, window, sinks, q_lens, kv_lens
    (1, 1, 1, 1, 1, 8, None, 0, None, None),                       # one token
    (2, 1, 300, 4, 2, 32, 40, 3, None, [300, 7]),                  # decoding: keys split between wavefronts and workgroups
    (1, 1, 70, 8, 1, 64, None, 0, None, None),
    (1, 37, 37, 2, 2, 40, None, 0, None, None),                    # odd size, padded head
    (2, 50, 50, 3, 1, 16, 9, 2, [50, 23], [50, 23]),               # padded batch
    (1, 40, 200, 4, 2, 96, 30, 35, None, None),                    # chunk over a cache; sinks longer than the window
    (2, 5, 60, 5, 1, 24, 1, 0, [5, 0], [3, 60]),                   # window of one; rows before the first key; no rows
    (1, 150, 150, 1, 1, 128, 20, 1, None, None),
    (2, 70, 70, 2, 1, 32, 13, 2, [-5, 999], [70, 999]),            # lengths outside the range are taken into it
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_and_gradients_in_emulation(seq, case, dtype):
    B, Nq, Nk, Hq, Hkv, D, window, sinks, ql, kl = ATTENTION[case]
    q, k, v, dout = ref.make_attention(B, Nq, Nk, Hq, Hkv, D, dtype, case, "cpu", by=2.0)
    kw = dict(window=window, sinks=sinks, q_lens=None if ql is None else torch.tensor(ql), kv_lens=None if kl is None else torch.tensor(kl))
    want = ref.attention(q, k, v, dout, **kw)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    ref.check((out, lse), want, ("out", "lse"))
    ref.check(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), want, ("dq", "dk", "dv"))


def test_attention_splits_the_rows_of_sinks_in_emulation(seq):
    q, k, v, dout = ref.make_attention(1, 600, 600, 1, 1, 16, "fp32", 5, "cpu")
    kw = dict(window=4, sinks=130)                                  # two tiles of sink keys, four parts of rows
    want = ref.attention(q, k, v, dout, **kw)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, **kw), want, ("out", "lse", "dq", "dk", "dv"))


LINEAR = [
    # B, N, H, Dk, Dv, decays, lens, state
    (1, 1, 1, 8, 8, [-0.1], None, True),
    (2, 70, 2, 32, 40, [0.0, -3.0], [70, 33], True),                # no decay, strong decay
    (1, 130, 2, 64, 32, [-0.02, float("-inf")], None, False),       # only the token itself
    (3, 65, 1, 16, 96, [-0.5], [0, 65, 64], True),                  # no tokens; a length at the chunk's end
    (1, 100, 1, 128, 128, [-0.01], None, True),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(LINEAR)))
def test_linear_attention_and_gradients_in_emulation(seq, case, dtype):
    B, N, H, Dk, Dv, g, lens, state = LINEAR[case]
    q, k, v, dout, s0, ds = ref.make_linear(B, N, H, Dk, Dv, dtype, case, "cpu", state)
    g = torch.tensor(g)
    lens = None if lens is None else torch.tensor(lens)
    want = ref.linear(q, k, v, g, dout, ds, initial=s0, lens=lens)
    ref.check(seq.linear_attention(q, k, v, g, initial_state=s0, lens=lens), want, ("out", "final"))
    ref.check(seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=lens), want, ("dq", "dk", "dv", "dinitial"))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_linear_attention_in_segments_in_emulation(seq, dtype):
    """Long enough for two segments: moments, scan and walk."""
    q, k, v, dout, s0, ds = ref.make_linear(1, 1100, 1, 8, 8, dtype, 3, "cpu")
    g = torch.tensor([-0.003])
    want = ref.linear(q, k, v, g, dout, ds, initial=s0)
    ref.check(seq.linear_attention(q, k, v, g, initial_state=s0), want, ("out", "final"))
    ref.check(seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0), want, ("dq", "dk", "dv", "dinitial"))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_linear_attention_of_many_heads_in_emulation(seq, dtype):
    """Enough heads that each is walked in one piece, which then forms the final moments too."""
    B, H = 18, 10
    q, k, v, dout, s0, ds = ref.make_linear(B, 90, H, 8, 8, dtype, 3, "cpu")
    g = -torch.rand(H, generator=torch.Generator().manual_seed(2))
    lens = torch.tensor([(7 * b) % 91 for b in range(B)])
    want = ref.linear(q, k, v, g, dout, ds, initial=s0, lens=lens)
    ref.check(seq.linear_attention(q, k, v, g, initial_state=s0, lens=lens), want, ("out", "final"))
    ref.check(seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=lens), want, ("dq", "dk", "dv", "dinitial"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Dk,Dv", [(8, 8), (32, 96), (128, 128)])
def test_step_goes_on_from_the_state_in_emulation(seq, dtype, Dk, Dv):
    q, k, v, _, s0, _ = ref.make_linear(2, 5, 3, Dk, Dv, dtype, 9, "cpu")
    g = torch.tensor([0.0, -0.3, float("-inf")])
    want = ref.linear(q, k, v, g, initial=s0)
    state = s0.clone()
    outs = [seq.linear_attention_step(q[:, t], k[:, t], v[:, t], g, state) for t in range(5)]
    ref.check((torch.stack(outs, 1), state), want, ("out", "final"))


def test_autograd_gives_the_gradients_in_emulation(seq):
    """Gradients of shared heads and of broadcast inputs; against differences of the definition."""
    q, k, v, dout = ref.make_attention(2, 9, 9, 4, 2, 16, "fp32", 1, "cpu")
    k1 = k[:1].clone().requires_grad_()                             # one sequence's keys for the whole batch
    q.requires_grad_()
    out = seq.window_attention(q, k1.expand(2, -1, -1, -1), v, window=4, sinks=1)
    dq, dk = torch.autograd.grad(out, (q, k1), dout)
    want = ref.attention(q, k1.expand(2, -1, -1, -1), v, dout, window=4, sinks=1)
    ref.check((dq,), want, ("dq",))
    total, bound = want["dk"][0].sum(0, keepdim=True), want["dk"][1].sum(0, keepdim=True)
    ref.check((dk,), {"dk": (total, bound + 2 * ref.W * total.abs())}, ("dk",))
    # directional differences of the 64-bit definition: the formula's gradient is the gradient
    e = 1e-6
    d = torch.randn(k1.shape, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    f = lambda s: float((ref.attention(q.detach().double(), (k1.detach().double() + s * d).expand(2, -1, -1, -1), v.double(), window=4,  # noqa: E731
                                       sinks=1)["out"][0] * dout.double()).sum())
    assert abs((f(e) - f(-e)) / (2 * e) - float((total * d).sum())) < 1e-6 * float((total * d).abs().sum())
    # the state's gradient comes back, in its own type
    q, k, v, dout, s0, ds = ref.make_linear(1, 6, 2, 8, 8, "fp32", 2, "cpu")
    s0 = s0.double().requires_grad_()
    g = torch.tensor([-0.1, -0.2])
    out, last = seq.linear_attention(q, k, v, g, initial_state=s0)
    (d0,) = torch.autograd.grad((out * dout).sum() + (last * ds).sum(), (s0,))
    assert d0.dtype == torch.float64
    ref.check((d0,), ref.linear(q, k, v, g, dout, ds, initial=s0), ("dinitial",))
    # only the state is used
    q.requires_grad_()
    k.requires_grad_()
    _, last = seq.linear_attention(q, k, v, g)
    dq, dk = torch.autograd.grad(last, (q, k), ds)
    want = ref.linear(q, k, v, g, torch.zeros_like(v), ds)
    ref.check((dq, dk), want, ("dq", "dk"))


def test_strides_orders_and_alignment_in_emulation(seq):
    """Any layout gives the bits of a contiguous copy."""
    q, k, v, dout = ref.make_attention(2, 20, 20, 4, 2, 32, "bf16", 6, "cpu")
    kw = dict(window=7, sinks=2)
    want, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    grads = seq.window_attention_grad(q, k, v, want, lse, dout, **kw)
    forms = {
        "heads first": lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
        "batch inside": lambda x: x.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3),
        "head size outside": lambda x: x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1),
        "odd rows": lambda x: torch.cat([x, x[..., :3]], 3)[..., :32],
        "odd start": lambda x: torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape),
        "reversed copy": lambda x: x.flip(1).flip(1),
    }
    for name, f in forms.items():
        assert torch.equal(f(q), q), name
        out, l2 = seq.window_attention(f(q), f(k), f(v), return_lse=True, **kw)
        assert torch.equal(out, want) and torch.equal(l2, lse), name
        for x, y in zip(seq.window_attention_grad(f(q), f(k), f(v), f(want), lse, f(dout), **kw), grads):
            assert torch.equal(x, y), name
    one = seq.window_attention(q[:, -1:], k, v, **kw)               # a slice of rows: the last token alone
    ref.check((one,), ref.attention(q[:, -1:], k, v, **kw), ("out",))


def test_what_lies_outside_the_lengths_is_not_read_in_emulation(seq):
    nan = float("nan")
    q, k, v, dout = ref.make_attention(2, 40, 40, 2, 1, 16, "fp32", 8, "cpu")
    lens = torch.tensor([40, 17])
    kw = dict(window=6, sinks=1, q_lens=lens, kv_lens=lens)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    grads = seq.window_attention_grad(q, k, v, out, lse, dout, **kw)
    for x in (q, k, v, dout):
        x[1, 17:] = nan
    out2, lse2 = seq.window_attention(q, k, v, return_lse=True, **kw)
    assert torch.equal(out, out2) and torch.equal(lse, lse2) and not out2[1, 17:].any()
    for x, y in zip(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), grads):
        assert torch.equal(x, y) and torch.isfinite(x).all()
    # keys before all windows, in the gradients too
    q, k, v, dout = ref.make_attention(1, 3, 300, 2, 1, 16, "fp32", 8, "cpu")
    kw = dict(window=5, sinks=2)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    grads = seq.window_attention_grad(q, k, v, out, lse, dout, **kw)
    k[:, 2:293], v[:, 2:293] = nan, nan                              # the first row stands at 297 and sees 293 .. 297
    for x, y in zip(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), grads):
        assert torch.equal(x, y) and torch.isfinite(x).all()
    assert not grads[1][:, 2:293].any() and grads[1][:, 293].any()
    # keys before the window of a single token
    q, k, v, _ = ref.make_attention(1, 1, 50, 2, 1, 16, "fp32", 8, "cpu")
    one = seq.window_attention(q, k, v, window=5, sinks=2)
    k[:, 2:45], v[:, 2:45] = nan, nan
    assert torch.equal(seq.window_attention(q, k, v, window=5, sinks=2), one)
    q, k, v, dout, s0, ds = ref.make_linear(2, 40, 1, 8, 8, "fp32", 8, "cpu")
    g, lens = torch.tensor([-0.1]), torch.tensor([40, 9])
    out, last = seq.linear_attention(q, k, v, g, initial_state=s0, lens=lens)
    grads = seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=lens)
    for x in (q, k, v, dout):
        x[1, 9:] = nan
    out2, last2 = seq.linear_attention(q, k, v, g, initial_state=s0, lens=lens)
    assert torch.equal(out, out2) and torch.equal(last, last2)
    for x, y in zip(seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0, lens=lens), grads):
        assert torch.equal(x, y)


def test_scale_of_either_sign_and_zero_in_emulation(seq):
    q, k, v, dout = ref.make_attention(1, 20, 30, 2, 1, 16, "fp32", 8, "cpu", by=3.0)
    for scale in (-0.7, 0.0, 1e-3, 2.0):
        want = ref.attention(q, k, v, dout, window=9, sinks=2, scale=scale)
        out, lse = seq.window_attention(q, k, v, window=9, sinks=2, scale=scale, return_lse=True)
        ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, window=9, sinks=2, scale=scale), want, ("out", "lse", "dq", "dk", "dv"))
    x, y, w, do, s0, ds = ref.make_linear(1, 20, 1, 8, 8, "fp32", 8, "cpu")
    g = torch.tensor([-0.2])
    want = ref.linear(x, y, w, g, do, ds, scale=-0.7, initial=s0)
    ref.check(seq.linear_attention(x, y, w, g, scale=-0.7, initial_state=s0) + seq.linear_attention_grad(x, y, w, g, do, ds, scale=-0.7, initial_state=s0),
              want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_empty_batches_and_lengths_in_emulation(seq):
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    for B, Nq, Nk in ((0, 3, 3), (2, 0, 3), (2, 3, 0), (1, 0, 0)):
        q, k = f(B, Nq, 2, 16), f(B, Nk, 1, 16)
        out, lse = seq.window_attention(q, k, k, window=2, sinks=1, return_lse=True)
        assert out.shape == q.shape and not out.any() and (lse == float("-inf")).all()
        for x, y in zip(seq.window_attention_grad(q, k, k, out, lse, q, window=2, sinks=1), (q, k, k)):
            assert x.shape == y.shape and not x.any()
    g = torch.tensor([-0.1, -0.2])
    for B, N in ((0, 3), (2, 0)):
        x, s = f(B, N, 2, 16), torch.randn(B, 2, 16, 16)
        out, last = seq.linear_attention(x, x, x, g, initial_state=s)
        assert out.shape == x.shape and torch.equal(last, s)
        dq, dk, dv, d0 = seq.linear_attention_grad(x, x, x, g, x, s, initial_state=s)
        assert dq.shape == x.shape and torch.equal(d0, s)
    assert seq.linear_attention_step(f(0, 2, 16), f(0, 2, 16), f(0, 2, 16), g, f(0, 2, 16, 16)).shape == (0, 2, 16)


def test_far_rows_and_many_shared_heads_in_emulation(seq):
    """Strides beyond the 32-bit offsets of the fast loads, overlapping rows, more query heads on one key head than a turn of a tile's loads has rows."""
    far = torch.randn(36 * (1 << 21), generator=torch.Generator().manual_seed(1))           # 8 MiB from token to token
    k = far.as_strided((1, 36, 1, 8), (far.numel(), 1 << 21, 8, 1))
    v = far[8:].as_strided((1, 36, 1, 8), (far.numel(), 1 << 21, 8, 1))
    q, _, _, dout = ref.make_attention(1, 36, 36, 2, 1, 8, "fp32", 8, "cpu")
    cases = [(q, k, v, dout), (q, k[:, 3:4].expand(1, 36, 1, 8), v, dout), ref.make_attention(1, 3, 40, 80, 1, 8, "fp32", 9, "cpu"),
             ref.make_attention(1, 40, 40, 6, 2, 8, "fp32", 9, "cpu")]
    for q, k, v, dout in cases:
        want = ref.attention(q, k, v, dout, window=7, sinks=2)
        out, lse = seq.window_attention(q, k, v, window=7, sinks=2, return_lse=True)
        ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, window=7, sinks=2), want, ("out", "lse", "dq", "dk", "dv"))
    far = torch.randn(5 * (1 << 23), generator=torch.Generator().manual_seed(1))            # 32 MiB
    x, y, w = (far[8 * i:].as_strided((1, 5, 1, 8), (far.numel(), 1 << 23, 8, 1)) for i in range(3))
    g = torch.tensor([-0.3])
    want = ref.linear(x, y, w, g, w)
    ref.check(seq.linear_attention(x, y, w, g) + seq.linear_attention_grad(x, y, w, g, w), want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_refusals_of_the_front_end(seq):
    f = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)  # noqa: E731
    q, k = f(2, 4, 4, 16), f(2, 6, 2, 16)
    ok = lambda **kw: seq.window_attention(q, k, k, **kw)  # noqa: E731
    ok()
    for bad in (dict(window=0), dict(sinks=-1), dict(scale=float("nan")), dict(q_lens=torch.zeros(3, dtype=torch.int32)),
                dict(kv_lens=torch.zeros(2)), dict(kv_lens=[1, 2])):
        with pytest.raises(AssertionError):
            ok(**bad)
    for a in ((q[0], k, k), (q, k[:1], k[:1]), (q, k, k[:, :5]), (q, k[..., :8], k), (q.double(), k.double(), k.double()),
              (q, k.half(), k), (f(2, 4, 3, 16), k, k)):
        with pytest.raises(AssertionError):
            seq.window_attention(*a)
    for d in (4, 12, 136):
        with pytest.raises(capi.F3MError) as e:
            seq.window_attention(f(1, 2, 1, d), f(1, 2, 1, d), f(1, 2, 1, d))
        assert e.value.code == 2
    out, lse = ok(return_lse=True)
    with pytest.raises(AssertionError):
        seq.window_attention_grad(q, k, k, out, lse.double(), out)
    with pytest.raises(AssertionError):
        seq.window_attention_grad(q, k, k, out, lse, out[:, :3])
    x, v, g = f(2, 4, 3, 16), f(2, 4, 3, 8), f(3)
    seq.linear_attention(x, x, v, g)
    for a, kw in (((x, x[:, :3], v, g), {}), ((x, x, v[:1], g), {}), ((x, x, v, f(2)), {}), ((x, x, v, g), dict(scale=0.0)),
                  ((x, x, v, g), dict(initial_state=f(2, 3, 8, 16))), ((x, x, v, g), dict(lens=f(2))), ((x, x, v, g.clone().requires_grad_()), {})):
        with pytest.raises(AssertionError):
            seq.linear_attention(*a, **kw)
    s = f(2, 3, 16, 8)
    y, w = f(2, 3, 16), f(2, 3, 8)
    seq.linear_attention_step(y, y, w, g, s)
    for a in ((y, y, w, g, s.double()), (y, y, w, g, s[:1]), (y, y, w, g, s.transpose(2, 3).contiguous().transpose(2, 3)),
              (x, x, v, g, s), (y.clone().requires_grad_(), y, w, g, s)):
        with pytest.raises(AssertionError):
            seq.linear_attention_step(*a)


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError):
        sequence.window_attention(x, x, x)
    with pytest.raises(RuntimeError):
        sequence.linear_attention(x, x, x, torch.zeros(1))
    with pytest.raises(RuntimeError):
        sequence.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(1), torch.zeros(1, 1, 8, 8))


def test_refusals_of_the_c_abi(emu_lib):
    lib = emu_lib
    buf = torch.zeros(4096, dtype=torch.float32)
    at = buf.data_ptr() + (-buf.data_ptr()) % 64
    ok = dict(dtype=2, D=8, Hq=2, Hkv=1, B=1, Nq=2, Nk=3, q0=32, q1=16, q2=8, k0=24, k1=8, k2=8, v0=24, v1=8, v2=8, window=0, sinks=0, scale=1.0)

    def attention(q=at, k=at, v=at, out=at + 4096, ws=at + 8192, size=8192, **kw):
        return lib.f3m_window_attention(C.byref(capi.AttnParams(**dict(ok, **kw))), q, k, v, None, None, out, None, ws, size, None)

    assert attention() == 0
    assert attention(D=12) == 2 and attention(Hq=3, Hkv=2) == 3 and attention(B=-1) == 3 and attention(dtype=7) == 61
    assert attention(window=-1) == 61 and attention(scale=float("inf")) == 61 and attention(Nk=1 << 40) == 3
    assert attention(q=None) == 8 and attention(out=None) == 8 and attention(k=at + 4) == 60 and attention(v1=9) == 60
    assert b"16 bytes" in lib.f3m_last_error()
    big = dict(Nq=1, Nk=4000)
    n = C.c_size_t()
    assert lib.f3m_window_attention_workspace(C.byref(capi.AttnParams(**dict(ok, **big))), 0, C.byref(n)) == 0 and n.value > 0
    assert attention(ws=at, size=n.value - 1, **big) == 62 and attention(ws=None, size=n.value, **big) == 8
    assert lib.f3m_window_attention_workspace(None, 0, C.byref(n)) == 8 and lib.f3m_window_attention_workspace(C.byref(capi.AttnParams(**ok)), 0, None) == 8
    lin = dict(dtype=2, Dk=8, Dv=8, H=1, B=1, N=1, q0=8, q1=8, q2=8, k0=8, k1=8, k2=8, v0=8, v1=8, v2=8, scale=1.0)

    def step(state=at, g=at, **kw):
        return lib.f3m_linear_attention_step(C.byref(capi.LinearParams(**dict(lin, **kw))), at, at, at, g, state, at + 4096, None)

    assert step() == 0
    assert step(N=2) == 3 and step(Dv=132) == 2 and step(scale=0.0) == 61 and step(state=None) == 8 and step(g=None) == 8 and step(k0=6, B=1) == 60


def test_library_exports_the_sequence_products():
    import re
    from f3m_amd import _lib
    header = open(os.path.join(ROOT, "include", "f3m_sequence.h")).read()
    declared = set(re.findall(r"^int (f3m_[a-z0-9_]+)\(", header, re.M))
    assert declared == set(capi.SEQUENCE_SYMBOLS)
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built yet (python -m f3m_amd.build)")
    lib = C.CDLL(_lib.LIB_PATH)
    for name in declared:
        assert hasattr(lib, name), name
