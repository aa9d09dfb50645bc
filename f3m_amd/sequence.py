"""PyTorch-ROCm front end of the kernel products over sequences (include/f3m_sequence.h).

Where ``engine`` multiplies by a kernel matrix of points, these multiply by a kernel matrix of query and key vectors that
stand in an order:

* ``window_attention``: the exponential kernel over the last ``window`` positions and the first ``sinks`` ones, rows divided by
  their sums (a near field and a few fixed sources);
* ``linear_attention``: a separable kernel with a decay for each head, carried as moments; ``linear_attention_step`` is its
  single token.

Tensors are (batch, tokens, heads, head size), bfloat16, float16 or float32, on one HIP device; head sizes are multiples of 8 up
to 128.  Any strides are taken: a tensor whose last dimension is not contiguous, or whose rows do not start at multiples of
16 bytes, is copied first.  Calls are queued on the current stream of the tensors' device and not waited for, allocate through
torch only, and can be captured into a graph.  Both products are differentiable once, backwards; forward-mode derivatives and tracing
are refused.  A captured step runs its backward pass inside the capture too, with no eager autograd graph of the same leaves alive, or calls the
``_grad`` functions, which keep no graph.

Values must be finite where a sequence has tokens; what lies behind its length is not read."""
import ctypes as C
import functools
import math
import operator

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib, capi
from .engine import _need_cuda, _prep

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _call(device, name, *args):
    """Queues a library call on the current stream of `device`."""
    lib, index = _lib.get(), device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = getattr(lib, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, stream)
    if rc:
        capi.check(lib, rc)


def _eager(*tensors):
    """The library reads memory and knows nothing of a derivative carried along or of a graph under construction, which would lose the call without a word."""
    if forward_ad._current_level >= 0 and any(torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the products over sequences have no forward-mode derivatives")
    if torch._C._is_tracing() or (torch._C._len_torch_dispatch_stack() and _proxy_mode()):
        raise RuntimeError("the products over sequences cannot be traced")


def _proxy_mode():
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def _workspace_bytes(name, params, grad):
    lib, n = _lib.get(), C.c_size_t()
    capi.check(lib, getattr(lib, name)(params, grad, C.byref(n)))
    return n.value


def _scratch(device, n):
    """Scratch memory of one call: torch's allocator hands it out in the order of the stream, a capture from the graph's own pool."""
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _strides(shape, stride, e):
    """Strides of all dimensions but the last for tensors of e bytes an element whose rows can be read 16 bytes at a time, else None.
    The stride of a dimension of one element is never used and may be anything."""
    if stride[-1] != 1 and shape[-1] != 1:
        return None
    s = [x if d > 1 else 0 for x, d in zip(stride[:-1], shape[:-1])]
    return None if any(x * e % 16 for x in s) else s


def _copy(t):
    return t.clone(memory_format=torch.contiguous_format)


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _check(ok, text):
    if not ok:
        raise AssertionError(text)


def _same(first, *others):
    d = first.get_device()
    for t in others:
        if t.get_device() != d:
            _need_cuda(first, *others)
            raise RuntimeError("tensors of one call must be on one device (got %s and %s)" % (first.device, t.device))
    if d < 0:
        _need_cuda(first)


def _lens(lens, B, like, name, most):
    if lens is None:
        return None
    _check(torch.is_tensor(lens) and lens.shape == (B,) and lens.dtype in (torch.int32, torch.int64),
           "%s must be an integer tensor of shape (%d,)" % (name, B))
    _same(like, lens)
    return _prep(lens if lens.dtype == torch.int32 else lens.clamp(0, most), torch.int32)        # the library takes values into the range, but after 32 bits


# ---- attention with a window and sinks --------------------------------------------------------------

@functools.lru_cache(maxsize=512)
def _attention_shape(dtype, q, qs, k, ks, v, vs, ds, window, sinks, scale, grad):
    """Checks of shapes and strides, and what the library needs to know of them: (parameters, bytes of workspace), or None where
    a tensor has to be copied first.  Kept by shape, not by tensor."""
    _check(len(q) == 4 and len(k) == 4 and len(v) == 4, "q, k and v must be (batch, tokens, heads, head size)")
    _check(dtype in _TYPES, "q, k and v must have one type: bfloat16, float16 or float32")
    B, Nq, Hq, D = q
    _check(k == v and k[0] == B and k[3] == D, "shapes of q, k and v do not match")
    Nk, Hkv = k[1], k[2]
    _check(Hq >= 1 and Hkv >= 1 and Hq % Hkv == 0, "the heads of q must be a multiple of those of k and v")
    _check(window is None or window >= 1, "window must be at least 1, or None for all positions")
    _check(sinks >= 0, "sinks must not be negative")
    window, sinks = min(window or 0, 1 << 62), min(sinks, 1 << 62)       # ctypes would cut what is beyond 64 bits; all positions either way
    scale = max(1, D) ** -0.5 if scale is None else scale
    _check(math.isfinite(scale), "scale must be finite")
    e = dtype.itemsize
    s = [_strides(x, y, e) for x, y in ((q, qs), (k, ks), (v, vs), (q, ds)) if y is not None]
    params = lambda s: capi.AttnParams(_TYPES[dtype], D, Hq, Hkv, B, Nq, Nk, *s, window, sinks, scale)  # noqa: E731
    if None in s:
        _workspace_bytes("f3m_window_attention_workspace", params([0] * 12), grad)       # shapes that no copy makes right are refused
        return None
    p = params(sum(s, []) + ([0, 0, 0] if ds is None else []))
    return p, _workspace_bytes("f3m_window_attention_workspace", p, grad)


def _attention_params(q, k, v, window, sinks, scale, dout=None):
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise AssertionError("q, k and v must be tensors")
    _same(q, k, v)
    t = q.dtype
    if k.dtype != t or v.dtype != t:
        raise AssertionError("q, k and v must have one type: bfloat16, float16 or float32")
    if dout is not None:
        _check(torch.is_tensor(dout) and dout.shape == q.shape, "dout must have the shape of out")
        _same(q, dout)
        if dout.dtype != t:
            dout = dout.to(t)
        if dout.data_ptr() % 16:
            dout = _copy(dout)
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        q, k, v = (_copy(x) if x.data_ptr() % 16 else x for x in (q, k, v))
    if type(window) is not int or type(sinks) is not int:
        window, sinks = None if window is None else operator.index(window), operator.index(sinks)
    if scale is not None:
        scale = float(scale)
    for _ in range(2):
        how = _attention_shape(t, q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), None if dout is None else dout.stride(),
                               window, sinks, scale, dout is not None)
        if how is not None:
            break
        q, k, v, dout = (x if x is None or _strides(x.shape, x.stride(), x.element_size()) else _copy(x) for x in (q, k, v, dout))
    return how[0], how[1], q, k, v, dout


def _attention(q, k, v, window, sinks, scale, q_lens, kv_lens, want_lse):
    p, n, q, k, v, _ = _attention_params(q, k, v, window, sinks, scale)
    if q_lens is not None:
        q_lens = _lens(q_lens, q.shape[0], q, "q_lens", q.shape[1])
    if kv_lens is not None:
        kv_lens = _lens(kv_lens, q.shape[0], q, "kv_lens", k.shape[1])
    d = q.device
    out = _like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=d) if want_lse else None
    ws = _scratch(d, n)
    _call(d, "f3m_window_attention", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_lens), _ptr(kv_lens), out.data_ptr(), _ptr(lse),
          _ptr(ws), n)
    return out, lse


def window_attention_grad(q, k, v, out, lse, dout, window=None, sinks=0, scale=None, q_lens=None, kv_lens=None):
    """(dq, dk, dv): gradients of sum(out * dout), from the out and lse that window_attention(..., return_lse=True)
    gave for the same arguments."""
    _eager(q, k, v, out, lse, dout)
    p, n, q, k, v, dout = _attention_params(q, k, v, window, sinks, scale, dout)
    _same(q, out, lse)
    _check(out.shape == q.shape and out.dtype == q.dtype, "out must have the shape and type of q")
    _check(lse.shape == q.shape[:3] and lse.dtype == torch.float32, "lse must be float32 (batch, tokens, heads)")
    q_lens, kv_lens = _lens(q_lens, q.shape[0], q, "q_lens", q.shape[1]), _lens(kv_lens, q.shape[0], q, "kv_lens", k.shape[1])
    out, lse = out.contiguous(), lse.contiguous()
    if out.data_ptr() % 16:
        out = out.clone()
    dq, dk, dv = _like(q), _like(k), _like(v)
    ws = _scratch(q.device, n)
    _call(q.device, "f3m_window_attention_grad", p, _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(dout), _ptr(q_lens),
          _ptr(kv_lens), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), n)
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, q_lens, kv_lens):
        out, lse = _attention(q, k, v, window, sinks, scale, q_lens, kv_lens, True)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, kv_lens)
        ctx.how = (window, sinks, scale)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 8
        q, k, v, out, lse, q_lens, kv_lens = ctx.saved_tensors
        return window_attention_grad(q, k, v, out, lse, dout, *ctx.how, q_lens, kv_lens) + (None,) * 5


def window_attention(q, k, v, window=None, sinks=0, scale=None, q_lens=None, kv_lens=None, return_lse=False):
    """Attention of q (B, Nq, Hq, D) to k, v (B, Nk, Hkv, D); query head h reads key head h // (Hq // Hkv).

    Row i of sequence b stands at position kv_lens[b] - q_lens[b] + i: the rows are the last tokens of the keys (one row and a
    long cache: a decoding step; a chunk of rows: a piece of a prompt; q_lens = kv_lens: a padded batch).  It sees the keys at
    positions up to its own that are among the last `window` (None: all) or the first `sinks`.  q_lens, kv_lens: integer tensors
    (B,), None for Nq and Nk; values are taken into that range.  scale: default D**-0.5.  Rows behind q_lens[b] and rows that see no key give 0.
    -> out (B, Nq, Hq, D), or (out, lse) with lse (B, Nq, Hq) float32, the logarithm of each row's sum (-inf: sees none; no gradient)."""
    _eager(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttention.apply(q, k, v, window, sinks, scale, q_lens, kv_lens)
    else:
        out, lse = _attention(q, k, v, window, sinks, scale, q_lens, kv_lens, return_lse)
    return (out, lse) if return_lse else out


# ---- linear attention with decays -------------------------------------------------------------------

def _decay(log_decay, H, like):
    if log_decay.dtype == torch.float32 and log_decay.shape == (H,) and log_decay.is_contiguous() and not log_decay.requires_grad:
        _same(like, log_decay)
        return log_decay
    _check(torch.is_tensor(log_decay) and log_decay.shape == (H,) and log_decay.is_floating_point(), "log_decay must be a float tensor of shape (%d,)" % H)
    _check(not (log_decay.requires_grad and torch.is_grad_enabled()), "log_decay is a constant: no gradient is computed for it")
    _same(like, log_decay)
    return _prep(log_decay, torch.float32)


def _state(state, shape, like, name):
    if state is None:
        return None
    _check(torch.is_tensor(state) and tuple(state.shape) == shape, "%s must be %s" % (name, shape))
    _same(like, state)
    return _prep(state, torch.float32)


@functools.lru_cache(maxsize=512)
def _linear_shape(dtype, q, qs, k, ks, v, vs, ds, scale, grad):
    """As _attention_shape; three dimensions: one token."""
    step = len(q) == 3
    _check(len(q) in (3, 4) and len(k) == len(q) and len(v) == len(q), "q, k and v must be (batch, tokens, heads, head size), or (batch, heads, head size) for a step")
    _check(dtype in _TYPES, "q, k and v must have one type: bfloat16, float16 or float32")
    _check(q == k and v[:-1] == q[:-1], "shapes of q, k and v do not match")
    B, H, Dk, Dv, N = q[0], q[-2], q[-1], v[-1], 1 if step else q[1]
    scale = max(1, Dk) ** -0.5 if scale is None else scale
    _check(math.isfinite(scale) and scale != 0, "scale must be finite and not 0")
    e = dtype.itemsize
    s = [_strides(x, y, e) for x, y in ((q, qs), (k, ks), (v, vs), (v, ds)) if y is not None]
    params = lambda s: capi.LinearParams(_TYPES[dtype], Dk, Dv, H, B, N, *s, scale)  # noqa: E731
    if None in s:
        _workspace_bytes("f3m_linear_attention_workspace", params([0] * 12), grad)
        return None
    if step:
        s = [[x[0], 0, x[1]] for x in s]
    p = params(sum(s, []) + ([0, 0, 0] if ds is None else []))
    return p, 0 if step else _workspace_bytes("f3m_linear_attention_workspace", p, grad)


def _linear_params(q, k, v, scale, dout=None, dims=4):
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise AssertionError("q, k and v must be tensors")
    _same(q, k, v)
    t = q.dtype
    if k.dtype != t or v.dtype != t:
        raise AssertionError("q, k and v must have one type: bfloat16, float16 or float32")
    _check(q.dim() == dims, "q must be (batch, tokens, heads, head size)" if dims == 4 else "q must be (batch, heads, head size)")
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        q, k, v = (_copy(x) if x.data_ptr() % 16 else x for x in (q, k, v))
    if dout is not None and dout.data_ptr() % 16:
        dout = _copy(dout)
    scale = None if scale is None else float(scale)
    for _ in range(2):
        how = _linear_shape(t, q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), None if dout is None else dout.stride(), scale,
                            dout is not None)
        if how is not None:
            break
        q, k, v, dout = (x if x is None or _strides(x.shape, x.stride(), x.element_size()) else _copy(x) for x in (q, k, v, dout))
    return how[0], how[1], q, k, v, dout


def _linear(q, k, v, log_decay, scale, initial_state, lens):
    p, n, q, k, v, _ = _linear_params(q, k, v, scale)
    (B, N, H, Dk), Dv = q.shape, v.shape[-1]
    g = _decay(log_decay, H, q)
    lens, initial_state = _lens(lens, B, q, "lens", N), _state(initial_state, (B, H, Dk, Dv), q, "initial_state")
    out = _like(v)
    final = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=q.device)
    ws = _scratch(q.device, n)
    _call(q.device, "f3m_linear_attention", p, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(initial_state), _ptr(lens), _ptr(out),
          _ptr(final), _ptr(ws), n)
    return out, final


def linear_attention_grad(q, k, v, log_decay, dout, dfinal_state=None, scale=None, initial_state=None, lens=None):
    """(dq, dk, dv, dinitial_state): gradients of sum(out * dout) + sum(final_state * dfinal_state)."""
    return _linear_grad(q, k, v, log_decay, dout, dfinal_state, scale, initial_state, lens, True)


def _linear_grad(q, k, v, log_decay, dout, dfinal_state, scale, initial_state, lens, want_initial):
    _eager(q, k, v, log_decay, dout, dfinal_state, initial_state)
    _check(torch.is_tensor(dout) and dout.shape == v.shape, "dout must have the shape of v")
    _same(q, dout)
    p, n, q, k, v, dout = _linear_params(q, k, v, scale, dout if dout.dtype == q.dtype else dout.to(q.dtype))
    (B, N, H, Dk), Dv = q.shape, v.shape[-1]
    g = _decay(log_decay, H, q)
    lens, initial_state = _lens(lens, B, q, "lens", N), _state(initial_state, (B, H, Dk, Dv), q, "initial_state")
    dfinal_state = _state(dfinal_state, (B, H, Dk, Dv), q, "dfinal_state")
    dq, dk, dv = _like(q), _like(k), _like(v)
    d0 = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=q.device) if want_initial else None
    ws = _scratch(q.device, n)
    _call(q.device, "f3m_linear_attention_grad", p, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(initial_state), _ptr(dout),
          _ptr(dfinal_state), _ptr(lens), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(d0), _ptr(ws), n)
    return dq, dk, dv, d0


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, lens):
        out, final = _linear(q, k, v, log_decay, scale, initial_state, lens)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, initial_state, lens = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 7
        if dout is None:
            dout = torch.zeros_like(v)
        want = ctx.needs_input_grad[5]
        dq, dk, dv, d0 = _linear_grad(q, k, v, log_decay, dout, dfinal, ctx.scale, initial_state, lens, want)
        return dq, dk, dv, None, None, d0.to(initial_state.dtype) if want else None, None


def linear_attention(q, k, v, log_decay, scale=None, initial_state=None, lens=None):
    """out_t = scale q_t^T S_t with S_t = exp(log_decay) S_{t-1} + k_t v_t^T, S_{-1} = initial_state (None: 0).

    q, k (B, N, H, Dk), v (B, N, H, Dv); log_decay (H,) float, at most 0, a constant; states (B, H, Dk, Dv) float32; scale: default
    Dk**-0.5.  lens: integer tensor (B,) or None; tokens behind lens[b] are not read, their out is 0.
    -> (out (B, N, H, Dv), final_state): the state after each sequence's last token, what a following call or
    linear_attention_step goes on from."""
    _eager(q, k, v, log_decay, initial_state)
    wants = [t for t in (q, k, v, initial_state) if torch.is_tensor(t) and t.requires_grad]
    if torch.is_grad_enabled() and wants:
        _check(not log_decay.requires_grad, "log_decay is a constant: no gradient is computed for it")
        return _LinearAttention.apply(q, k, v, log_decay, scale, initial_state, lens)
    return _linear(q, k, v, log_decay, scale, initial_state, lens)


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One token of linear_attention for each sequence: q, k (B, H, Dk), v (B, H, Dv) -> out (B, H, Dv).

    state (B, H, Dk, Dv), contiguous float32, becomes exp(log_decay) state + k v^T in place.  Not differentiable."""
    _eager(q, k, v, log_decay, state)
    _check(not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)),
           "linear_attention_step is not differentiable: use linear_attention")
    p, _, q, k, v, _ = _linear_params(q, k, v, scale, dims=3)
    (B, H, Dk), Dv = q.shape, v.shape[-1]
    g = _decay(log_decay, H, q)
    _same(q, state)
    _check(state.shape == (B, H, Dk, Dv) and state.dtype == torch.float32 and state.is_contiguous(),
           "state must be contiguous float32 %s" % ((B, H, Dk, Dv),))
    d = q.device
    out = _like(v)
    _call(d, "f3m_linear_attention_step", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), state.data_ptr(), out.data_ptr())
    increment_version(state)                                         # a product that kept it for its backward pass refuses that pass now
    return out
