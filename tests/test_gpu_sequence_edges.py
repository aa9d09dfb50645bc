"""GPU tests of the sequence products at the ends of their ranges."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import sequence_reference as ref  # noqa: E402
from test_gpu_sequence import ints, seq  # noqa: E402,F401


@pytest.mark.parametrize("Nk,window,kl", [(131300, None, [5]), (160600, 16, None)])
def test_gradients_of_tiles_that_no_row_sees(seq, Nk, window, kl):
    """Tiles of keys far behind a short sequence or far before the window, 16384 query heads on one key head: their row numbers lie beyond 32 bits."""
    print("case unseen tiles", Nk, window, kl, flush=True)
    G = 16384
    q, k, v, dout = ref.make_attention(1, 1, Nk, 1, 1, 8, "fp32", 3, "cuda")
    kw = dict(window=window, kv_lens=ints(kl))
    many = lambda x: x.expand(1, 1, G, 8)  # noqa: E731
    out, lse = seq.window_attention(many(q), k, v, return_lse=True, **kw)
    dq, dk, dv = seq.window_attention_grad(many(q), k, v, out, lse, many(dout), **kw)
    one = ref.attention(q, k, v, dout, **kw)
    for g in (0, G - 1):
        ref.check((out[:, :, g:g + 1], dq[:, :, g:g + 1]), one, ("out", "dq"))
    # every head alike: G times the gradients of one, a sum of G equal terms in fp32
    want = {n: (G * one[n][0], G * one[n][1] + (G + 32) * ref.W * G * one[n][0].abs()) for n in ("dk", "dv")}
    ref.check((dk, dv), want, ("dk", "dv"))
