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
