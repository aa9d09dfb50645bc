"""GPU tests of the products over sequences against their definitions in 64 bits (tests/sequence_reference.py, which derives the bounds)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import sequence_reference as ref  # noqa: E402


@pytest.fixture(scope="module")
def seq():
    assert torch.cuda.is_available(), "these tests need a GPU"
    from f3m_amd import _lib, sequence
    _lib.get()
    return sequence


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


ATTENTION = [
    # B, Nq, Nk, Hq, Hkv, D, window, sinks, q_lens, kv_lens
    (1, 1, 1, 1, 1, 8, None, 0, None, None),
    (2, 1, 2, 2, 1, 128, 1, 1, None, [2, 0]),
    (3, 1, 4097, 8, 2, 128, 700, 4, None, [4097, 1, 650]),          # decoding over caches of different lengths
    (1, 1, 5000, 16, 1, 64, None, 0, None, None),                   # 16 rows, one cache: split between workgroups
    (2, 3, 900, 40, 4, 96, 100, 5, None, [900, 2]),                  # 30 rows a head; fewer keys than rows
    (1, 7, 1300, 7, 1, 80, None, 0, None, None),                     # 49 rows: two wavefronts by two
    (2, 129, 1111, 6, 3, 104, 200, 70, None, [1111, 500]),           # a chunk over a cache; sinks longer than a tile
    (1, 333, 333, 5, 5, 72, None, 0, None, None),
    (2, 512, 512, 8, 1, 64, 64, 0, [512, 77], [512, 77]),
    (4, 200, 200, 3, 3, 32, 17, 2, [200, 0, 1, 199], [200, 0, 1, 199]),
    (1, 1000, 1000, 4, 2, 128, 50, 140, None, None),                 # two tiles of sinks, their rows in parts
    (1, 700, 700, 2, 2, 16, 1000, 3, None, None),                    # window longer than the sequence
    (4, 300, 300, 8, 4, 64, None, 0, [300, 20, 150, 299], [300, 20, 150, 299]),             # 16 pairs of sequence and head, two for each XCD
    (2, 300, 150, 2, 1, 128, 40, 2, None, None),                     # more rows than keys: the first see nothing
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_and_gradients(seq, case, dtype):
    B, Nq, Nk, Hq, Hkv, D, window, sinks, ql, kl = ATTENTION[case]
    print("case attention", ATTENTION[case], dtype, flush=True)
    q, k, v, dout = ref.make_attention(B, Nq, Nk, Hq, Hkv, D, dtype, case, "cuda", by=2.0)
    kw = dict(window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kl))
    want = ref.attention(q, k, v, dout, **kw)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    ref.check((out, lse), want, ("out", "lse"))
    grads = seq.window_attention_grad(q, k, v, out, lse, dout, **kw)
    ref.check(grads, want, ("dq", "dk", "dv"))
    # the same bits again
    assert torch.equal(seq.window_attention(q, k, v, **kw), out)
    for x, y in zip(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), grads):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 96, 128])
def test_attention_of_every_head_size(seq, D, dtype):
    print("case head size", D, dtype, flush=True)
    for Nq, Nk, G in ((150, 150, 1), (2, 400, 4), (12, 300, 5)):
        q, k, v, dout = ref.make_attention(1, Nq, Nk, 2 * G, 2, D, dtype, D, "cuda")
        kw = dict(window=60, sinks=3)
        want = ref.attention(q, k, v, dout, **kw)
        out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
        ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, **kw), want, ("out", "lse", "dq", "dk", "dv"))


def test_large_logits(seq):
    """Logits of several hundreds of either sign: one key takes nearly all of a row."""
    q, k, v, dout = ref.make_attention(1, 100, 100, 2, 2, 64, "bf16", 3, "cuda", by=60.0)
    want = ref.attention(q, k, v, dout)
    out, lse = seq.window_attention(q, k, v, return_lse=True)
    ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout), want, ("out", "lse", "dq", "dk", "dv"))
    q, k, v, _ = ref.make_attention(1, 3, 2000, 1, 1, 64, "fp16", 3, "cuda")
    k = -q[:, 2:3].expand_as(k) * 40                                 # every logit far below zero: the maximum is not 0
    out = seq.window_attention(q, k, v)
    ref.check((out,), ref.attention(q, k, v), ("out",))


def test_offsets_past_32_bits(seq):
    """A cache of 4.3 GB for k: one token at its end, the window, and the sinks at its start."""
    n, H, D = 4_200_000, 4, 128
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(1, n, H, D, generator=g, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(1, n, H, D, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(1, 2, H, D, generator=g, device="cuda", dtype=torch.bfloat16)
    out = seq.window_attention(q, k, v, window=300, sinks=4)
    # the same rows over the visible keys alone: 4 sinks and 301 positions; the sinks stay visible
    short = lambda x: torch.cat([x[:, :4], x[:, n - 301:]], 1)  # noqa: E731
    ref.check((out,), ref.attention(q, short(k), short(v), window=300, sinks=4), ("out",))
    assert torch.equal(out, seq.window_attention(q, short(k), short(v), window=300, sinks=4))


LINEAR = [
    # B, N, H, Dk, Dv, decays, lens, state
    (1, 1, 1, 8, 8, [-0.1], None, True),
    (2, 64, 2, 64, 64, [0.0, -3.0], [64, 63], True),
    (2, 333, 3, 128, 40, [-0.02, float("-inf"), -0.3], [333, 0], True),
    (1, 1000, 2, 96, 128, [-0.01, -1e-4], None, False),
    (3, 1500, 1, 128, 128, [-0.002], [1500, 1025, 511], True),       # segments; lengths at and beside their ends
    (1, 4100, 2, 32, 16, [0.0, -20.0], None, True),
    (60, 200, 3, 64, 32, [-0.1, -0.01, -0.5], [200 - 3 * b for b in range(60)], True),      # many heads: one walk each, final moments with it
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(LINEAR)))
def test_linear_attention_and_gradients(seq, case, dtype):
    B, N, H, Dk, Dv, g, lens, state = LINEAR[case]
    print("case linear", LINEAR[case], dtype, flush=True)
    q, k, v, dout, s0, ds = ref.make_linear(B, N, H, Dk, Dv, dtype, case, "cuda", state)
    g = torch.tensor(g, device="cuda")
    kw = dict(initial_state=s0, lens=ints(lens))
    want = ref.linear(q, k, v, g, dout, ds, initial=s0, lens=lens)
    got = seq.linear_attention(q, k, v, g, **kw)
    ref.check(got, want, ("out", "final"))
    grads = seq.linear_attention_grad(q, k, v, g, dout, ds, **kw)
    ref.check(grads, want, ("dq", "dk", "dv", "dinitial"))
    for x, y in zip(seq.linear_attention(q, k, v, g, **kw) + seq.linear_attention_grad(q, k, v, g, dout, ds, **kw), got + grads):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_linear_attention_of_every_head_size(seq, dtype):
    g = torch.tensor([-0.05, -0.5], device="cuda")
    for Dk in (8, 32, 64, 96, 128):
        for Dv in (24, 64, 88, 128):
            print("case head sizes", Dk, Dv, dtype, flush=True)
            q, k, v, dout, s0, ds = ref.make_linear(1, 100, 2, Dk, Dv, dtype, Dk + Dv, "cuda")
            want = ref.linear(q, k, v, g, dout, ds, initial=s0)
            ref.check(seq.linear_attention(q, k, v, g, initial_state=s0) + seq.linear_attention_grad(q, k, v, g, dout, ds, initial_state=s0),
                      want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_large_moments_in_half_precision(seq):
    """Without a decay the moments of 3000 like tokens pass fp16's largest number; out stays within it."""
    q, k, v, _, _, _ = ref.make_linear(1, 3000, 1, 64, 64, "fp16", 1, "cuda", False)
    k, v = k.abs() * 8 + 4, v.abs() * 4 + 4
    q = q * 0.01
    g = torch.zeros(1, device="cuda")
    want = ref.linear(q, k, v, g)
    assert float(want["final"][0].max()) > 65504
    ref.check(seq.linear_attention(q, k, v, g), want, ("out", "final"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_steps_go_on_from_a_prompt(seq, dtype):
    """A prompt, then single tokens on its final state: the values of the whole sequence."""
    q, k, v, _, _, _ = ref.make_linear(3, 140, 4, 128, 96, dtype, 5, "cuda", False)
    g = torch.tensor([-0.5, -0.05, -0.005, 0.0], device="cuda")
    want = ref.linear(q, k, v, g)
    out, state = seq.linear_attention(q[:, :135], k[:, :135], v[:, :135], g)
    outs = [seq.linear_attention_step(q[:, t], k[:, t], v[:, t], g, state) for t in range(135, 140)]
    ref.check((torch.cat([out, torch.stack(outs, 1)], 1), state), want, ("out", "final"))


def test_both_products_together_as_a_model_runs_them(seq):
    """A layer of each, trained: the gradients of the whole against 64 bits; then the same prompt served in a chunk and single tokens."""
    torch.manual_seed(0)
    B, N, H, D = 2, 150, 4, 64
    g = torch.tensor([-0.5, -0.1, -0.02, -0.004], device="cuda")
    x = torch.randn(B, N, H, 3 * D, device="cuda")

    def model(x, attention, linear):
        q, k, v = x.chunk(3, 3)
        y = attention(q, k[:, :, :2], v[:, :, :2])
        return linear(q, k * D ** -0.5, y)

    def attention64(q, k, v):
        see = ref.visible(N, N, 40, 2, "cuda")
        k, v = (t.repeat_interleave(H // t.shape[2], 2) for t in (k, v))
        s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
        return torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~see, float("-inf")), 3), v)

    def linear64(q, k, v):
        d = torch.arange(N, device="cuda")[:, None] - torch.arange(N, device="cuda")
        w = torch.exp(g.double()[:, None, None] * d.clamp(min=0)) * (d >= 0)
        return torch.einsum("bhij,bjhd->bihd", torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5 * w, v)

    y0 = x.double().requires_grad_()
    out0 = model(y0, attention64, linear64)
    (d0,) = torch.autograd.grad(out0.sum(), y0)
    y1 = x.clone().requires_grad_()
    out1 = model(y1, lambda q, k, v: seq.window_attention(q, k, v, window=40, sinks=2), lambda q, k, v: seq.linear_attention(q, k, v, g)[0])
    (d1,) = torch.autograd.grad(out1.sum(), y1)
    # two products in a row of fp32 sums of at most 150 x 64 terms: 2 x (150 + 64 + 100) x 2^-24 of the largest magnitudes
    for a, b in ((out1.detach(), out0.detach()), (d1, d0)):
        assert float((a.double() - b).abs().max()) < 2 * 314 * ref.W * 8 * float(b.abs().max())

    # served: 100 tokens in a chunk, then one at a time over a cache with room
    cache = torch.full((2, B, 160, 2, D), float("nan"), device="cuda")
    outs, state = [], None
    for a, b in [(0, 100)] + [(t, t + 1) for t in range(100, N)]:
        q, k, v = x[:, a:b].chunk(3, 3)
        cache[0, :, a:b], cache[1, :, a:b] = k[:, :, :2], v[:, :, :2]
        y = seq.window_attention(q, cache[0], cache[1], window=40, sinks=2, kv_lens=ints([b] * B))
        if state is None:
            o, state = seq.linear_attention(q, k * D ** -0.5, y, g)
        else:
            o = seq.linear_attention_step(q[:, 0], k[:, 0] * D ** -0.5, y[:, 0], g, state)[:, None]
        outs.append(o)
    assert float((torch.cat(outs, 1).double() - out0.detach()).abs().max()) < 2 * 314 * ref.W * 8 * float(out0.detach().abs().max())


def test_another_stream_and_back(seq):
    q, k, v, dout = ref.make_attention(2, 300, 300, 4, 2, 64, "bf16", 1, "cuda")
    want, lse = seq.window_attention(q, k, v, window=50, return_lse=True)
    grads = seq.window_attention_grad(q, k, v, want, lse, dout, window=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = q * 1.0                                                  # made on this stream: the call has to wait for it there
        out, l2 = seq.window_attention(a, k, v, window=50, return_lse=True)
        g2 = seq.window_attention_grad(a, k, v, out, l2, dout, window=50)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((want, lse) + grads, (out, l2) + g2):
        assert torch.equal(x, y)


def test_two_calls_at_once(seq):
    """Calls on two streams that overlap: each has its own workspace."""
    sets = [ref.make_attention(1, 4, 20000, 16, 2, 128, "bf16", n, "cuda") for n in (1, 2)]
    lin = [ref.make_linear(1, 3000, 4, 64, 64, "bf16", n, "cuda") for n in (1, 2)]
    g = torch.tensor([-0.5, -0.1, -0.01, -0.001], device="cuda")

    def call(n):
        q, k, v, _ = sets[n]
        x, y, w, dout, s0, ds = lin[n]
        return (seq.window_attention(q, k, v, window=15000, sinks=4),) + seq.linear_attention(x, y, w, g, initial_state=s0) + \
            seq.linear_attention_grad(x, y, w, g, dout, ds, initial_state=s0)

    want = [call(n) for n in (0, 1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(call(n))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for n in (0, 1):
        for r in got[n]:
            for a, b in zip(r, want[n]):
                assert torch.equal(a, b)


def test_captured_graphs_replay_beside_each_other(seq):
    """Two captured graphs with workspaces (split keys; segments), replayed in turn with eager work between, against eager results."""
    q, k, v, _ = ref.make_attention(1, 1, 6000, 8, 2, 128, "bf16", 1, "cuda")
    x, y, w, dout, s0, ds = ref.make_linear(1, 2100, 2, 64, 64, "bf16", 2, "cuda")
    g = torch.tensor([-0.1, -0.01], device="cuda")
    lens = ints([6000])

    def one():
        return (seq.window_attention(q, k, v, window=5000, sinks=4, kv_lens=lens),)

    def two():
        return seq.linear_attention(x, y, w, g, initial_state=s0) + seq.linear_attention_grad(x, y, w, g, dout, ds, initial_state=s0)

    graphs = []
    for f in (one, two):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = f()
        graphs.append((gr, out, f))
    for turn in range(4):
        q.normal_(generator=torch.Generator(device="cuda").manual_seed(turn))
        x.normal_(generator=torch.Generator(device="cuda").manual_seed(turn + 9))
        lens.fill_(6000 - 1700 * turn)
        for gr, out, f in graphs:
            for o in out:
                o.fill_(float("nan"))
            gr.replay()
        for gr, out, f in graphs:
            for a, b in zip(out, f()):
                assert torch.equal(a, b), turn


def test_a_training_step_in_a_graph(seq):
    q, k, v, dout = ref.make_attention(1, 200, 200, 4, 2, 64, "fp16", 1, "cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        return torch.autograd.grad(seq.window_attention(*leaves, window=30, sinks=2), leaves, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_host_and_mixed_tensors_are_refused(seq):
    x = torch.zeros(1, 2, 1, 8, device="cuda")
    with pytest.raises(RuntimeError):
        seq.window_attention(x, x.cpu(), x)
    with pytest.raises(RuntimeError):
        seq.window_attention(x, x, x, kv_lens=torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        seq.linear_attention(x, x, x, torch.zeros(1))
    from f3m_amd.capi import F3MError
    y = torch.zeros(1, 2, 1, 136, device="cuda")
    with pytest.raises(F3MError):
        seq.window_attention(y, y, y)


def test_scale_of_either_sign_and_zero(seq):
    q, k, v, dout = ref.make_attention(1, 120, 300, 2, 1, 64, "bf16", 8, "cuda", by=2.0)
    for scale in (-0.3, 0.0, 1e-3):
        want = ref.attention(q, k, v, dout, window=90, sinks=2, scale=scale)
        out, lse = seq.window_attention(q, k, v, window=90, sinks=2, scale=scale, return_lse=True)
        ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, window=90, sinks=2, scale=scale), want, ("out", "lse", "dq", "dk", "dv"))


def test_empty_batches_and_lengths(seq):
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    for B, Nq, Nk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k = f(B, Nq, 2, 16), f(B, Nk, 1, 16)
        out, lse = seq.window_attention(q, k, k, window=2, sinks=1, return_lse=True)
        assert not out.any() and (lse == float("-inf")).all()
        for x, y in zip(seq.window_attention_grad(q, k, k, out, lse, q, window=2, sinks=1), (q, k, k)):
            assert x.shape == y.shape and not x.any()
    x, s, g = f(2, 0, 2, 16), torch.randn(2, 2, 16, 16, device="cuda"), torch.tensor([-0.1, -0.2], device="cuda")
    out, last = seq.linear_attention(x, x, x, g, initial_state=s)
    assert out.shape == x.shape and torch.equal(last, s)
    assert torch.equal(seq.linear_attention_grad(x, x, x, g, x, s, initial_state=s)[3], s)


def test_far_rows_and_many_shared_heads(seq):
    far = torch.randn(36 * (1 << 22), device="cuda", dtype=torch.bfloat16)                  # 8 MiB from token to token
    k = far.as_strided((1, 36, 1, 64), (far.numel(), 1 << 22, 64, 1))
    v = far[64:].as_strided((1, 36, 1, 64), (far.numel(), 1 << 22, 64, 1))
    q, _, _, dout = ref.make_attention(1, 36, 36, 2, 1, 64, "bf16", 8, "cuda")
    cases = [(q, k, v, dout), (q, k[:, 3:4].expand(1, 36, 1, 64), v, dout), ref.make_attention(1, 3, 400, 80, 1, 64, "bf16", 9, "cuda"),
             ref.make_attention(1, 400, 400, 6, 2, 64, "bf16", 9, "cuda")]
    for n, (q, k, v, dout) in enumerate(cases):
        print("case far rows", n, flush=True)
        want = ref.attention(q, k, v, dout, window=70, sinks=2)
        out, lse = seq.window_attention(q, k, v, window=70, sinks=2, return_lse=True)
        ref.check((out, lse) + seq.window_attention_grad(q, k, v, out, lse, dout, window=70, sinks=2), want, ("out", "lse", "dq", "dk", "dv"))
    far = torch.randn(70 * (1 << 24), device="cuda", dtype=torch.bfloat16)                  # 32 MiB
    x, y, w = (far[64 * i:].as_strided((1, 70, 1, 64), (far.numel(), 1 << 24, 64, 1)) for i in range(3))
    y = y * 0.1
    g = torch.tensor([-0.3], device="cuda")
    want = ref.linear(x, y, w, g, w)
    ref.check(seq.linear_attention(x, y, w, g) + seq.linear_attention_grad(x, y, w, g, w), want, ("out", "final", "dq", "dk", "dv", "dinitial"))


def test_keys_before_all_windows_are_not_read(seq):
    nan = float("nan")
    q, k, v, dout = ref.make_attention(1, 3, 3000, 8, 2, 128, "bf16", 8, "cuda")
    kw = dict(window=500, sinks=2)
    out, lse = seq.window_attention(q, k, v, return_lse=True, **kw)
    grads = seq.window_attention_grad(q, k, v, out, lse, dout, **kw)
    k[:, 2:2498], v[:, 2:2498] = nan, nan                            # the first row stands at 2997 and sees 2498 .. 2997
    assert torch.equal(seq.window_attention(q, k, v, **kw), out)
    for x, y in zip(seq.window_attention_grad(q, k, v, out, lse, dout, **kw), grads):
        assert torch.equal(x, y)
