"""Operators over sequences of frames, next to the Savitzky-Golay filter (savgol_filer.py) and the per-frame ring of the
real-time tail (realtime.py): what a model over the tokens of a sequence -- frames, joints of frames, cells of feature maps or
of the voxel grid -- needs around its matrix products.  The reference has no such model; these have no counterpart in it.

    layer_norm               layer norm over the last axis
    rotate_positions         rotary positions with several axes (time, height, width; x, y, z) on q and k
    window_attention         attention with a sliding window and first tokens that stay visible, over recorded sequences
    window_cache_fill        fills the ring of a stream from a recorded sequence
    window_attention_step    the same attention for one new token per stream, over that ring

Tensors are float32, bfloat16 or float16 HIP tensors, tokens are (batch, tokens, heads, head_dim).  Arithmetic, sums and
softmax statistics are float32, results are rounded once to the input's type.  Calls are asynchronous on torch's current
stream of the tensors' device and can be captured into a graph.  layer_norm, rotate_positions and window_attention are
differentiable (once) by backward kernels whose sums run in a fixed order; inputs with forward-mode tangents are refused.
"""
import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from poseestimation_amd import _cabi

_DTYPES = {torch.float32: _cabi.F32, torch.bfloat16: _cabi.BF16, torch.float16: _cabi.F16}
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


# The smallest calls of this module take a few microseconds of GPU time, less than the checks of their arguments would when
# made one by one.  Each entry point therefore accepts the usual case by one cheap condition and looks for what is wrong, and
# how to say it, only where that fails.


def _check(t, name, like=None, like_name=None):
    """Raises unless `t` is a HIP tensor of an element type of this module (and of `like`'s type and device)."""
    if not torch.is_tensor(t):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(t).__name__))
    if not t.is_cuda:
        raise _cabi.MvxError("%s is on %s: the mvx kernels run on a HIP device only (no CPU path)" % (name, t.device))
    if t.dtype not in _DTYPES:
        raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if like is not None:
        if t.dtype != like.dtype:
            raise ValueError("%s is %s but %s is %s" % (name, t.dtype, like_name, like.dtype))
        if t.device != like.device:
            _cabi.same_device(like, like_name, **{name: t})


def _check_qkv(q, k, v):
    try:
        if q.is_cuda and q.dtype in _DTYPES and q.dtype == k.dtype == v.dtype and q.get_device() == k.get_device() == v.get_device():
            return
    except AttributeError:
        pass
    _check(q, "q")
    _check(k, "k", q, "q")
    _check(v, "v", q, "q")


_lib = None


def _run(index, what, entry, *args):
    """Calls the C entry point `entry` on torch's current stream of device `index`."""
    global _lib
    if _lib is None:
        _lib = _cabi.load()
    entry = getattr(_lib, entry)
    if index == torch.cuda.current_device():
        status = entry(*args, _cabi.raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _cabi.raw_stream(index))
    if status != _cabi.MVX_OK:
        _cabi.check(status, what)


def _pointer(t):
    return t.data_ptr() if t is not None else None


@functools.lru_cache(maxsize=1024)
def _int64s(values):
    return (ctypes.c_int64 * 4)(*values)


@functools.lru_cache(maxsize=1024)
def _int32s(values):
    return (ctypes.c_int32 * len(values))(*values)


def _strides(t):
    return _int64s(t.stride())


def _workspace(n_bytes, device):
    return torch.empty(max(n_bytes, 16), dtype=torch.uint8, device=device)


# ---- layer norm --------------------------------------------------------------------------------------------------------


def _norm_check(x, weight, bias, eps):
    _check(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("x must have a last axis of at least one value, got shape %s" % (tuple(x.shape),))
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative, got %r" % (eps,))
    param = weight if weight is not None else bias
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _check(p, name)
        _cabi.same_device(x, "x", **{name: p})
        if p.shape != x.shape[-1:]:
            raise ValueError("%s must have shape %s, got %s" % (name, tuple(x.shape[-1:]), tuple(p.shape)))
        if p.dtype not in (x.dtype, torch.float32) or p.dtype != param.dtype:
            raise ValueError("weight and bias must both be float32 or both of x's type %s, got %s for %s" % (x.dtype, p.dtype, name))


def _norm_usual(x, weight, bias, eps):
    """Whether this is a call with both parameters of x's type in which nothing is wrong."""
    try:
        width = x.shape[-1]
        return (x.is_cuda and weight.dtype == bias.dtype == x.dtype and x.dtype in _DTYPES and weight.shape == bias.shape == (width,)
                and x.get_device() == weight.get_device() == bias.get_device() and width > 0 and 0.0 <= eps < math.inf)
    except (AttributeError, IndexError, TypeError):
        return False


def _norm_run(x, weight, bias, eps, param_f32, want_stats):
    width = x.shape[-1]
    rows = x.numel() // width
    x = x.contiguous()
    y = torch.empty_like(x)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if want_stats else None
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    _run(x.get_device(), "layer_norm", "mvx_layer_norm", x.data_ptr(), _pointer(weight), _pointer(bias), _DTYPES[x.dtype],
         param_f32, rows, width, eps, y.data_ptr(), _pointer(stats))
    return x, y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, param_f32):
        x, y, stats = _norm_run(x, weight, bias, eps, param_f32, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_f32 = param_f32
        ctx.bias_like = None if bias is None else (bias.shape, bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, stats = ctx.saved_tensors
        width = x.shape[-1]
        rows = x.numel() // width
        grad_y = grad_y.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        weight = weight.contiguous() if weight is not None else None
        grad_x = torch.empty_like(x) if need_x else None
        grad_w = torch.empty(width, dtype=weight.dtype, device=x.device) if need_w else None
        grad_b = torch.empty(ctx.bias_like[0], dtype=ctx.bias_like[1], device=x.device) if need_b else None
        dtype = _DTYPES[x.dtype]
        n_bytes = _cabi.load().mvx_layer_norm_backward_workspace_bytes(dtype, rows, width) if need_w or need_b else 0
        ws = _workspace(n_bytes, x.device)
        _run(x.get_device(), "layer_norm", "mvx_layer_norm_backward", grad_y.data_ptr(), x.data_ptr(), _pointer(weight),
             stats.data_ptr(), dtype, ctx.param_f32, rows, width, _pointer(grad_x), _pointer(grad_w), _pointer(grad_b),
             ws.data_ptr(), ws.numel())
        return grad_x, grad_w, grad_b, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x (..., width) over its last axis: (x - mean) / sqrt(var + eps) * weight + bias, in x's type.

    weight and bias (width,) are of x's type or float32 (both alike); None stands for ones and zeros.  Differentiable with
    respect to x, weight and bias."""
    param_f32 = 0
    if not _norm_usual(x, weight, bias, eps):
        _norm_check(x, weight, bias, eps)
        param = weight if weight is not None else bias
        param_f32 = int(param is not None and param.dtype == torch.float32)
    _cabi.no_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and _cabi.needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps), param_f32)
    return _norm_run(x, weight, bias, eps, param_f32, False)[1]


# ---- rotary positions --------------------------------------------------------------------------------------------------


def _rotate_run(q, k, positions, sections, base, shared, pairs, inverse):
    b, n, heads, dim = q.shape
    if q.stride(3) != 1:
        q = q.contiguous()
    q_out = torch.empty((b, n, heads, dim), dtype=q.dtype, device=q.device)
    k_out, k_args = None, (None, None, 0)
    if k is not None:
        if k.stride(3) != 1:
            k = k.contiguous()
        k_heads = k.shape[2]
        k_out = torch.empty((b, n, k_heads, dim), dtype=q.dtype, device=q.device)
        k_args = (k.data_ptr(), _strides(k), k_heads)
    n_axes = len(sections)
    _run(q.get_device(), "rotate_positions", "mvx_rotate_positions", q.data_ptr(), _strides(q), heads, *k_args, _DTYPES[q.dtype], b, n,
         dim, positions.data_ptr(), _POSITION_TYPES[positions.dtype], n * n_axes if positions.dim() == 3 else 0, n_axes,
         _int32s(sections), base, shared, pairs, inverse, q_out.data_ptr(), _pointer(k_out))
    return q_out, k_out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base, shared, pairs):
        ctx.save_for_backward(positions)
        ctx.how = (sections, base, shared, pairs)
        ctx.with_k = k is not None
        return _rotate_run(q, k, positions, sections, base, shared, pairs, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        positions, = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[0], ctx.with_k and ctx.needs_input_grad[1]
        if need_q and need_k:
            grad_q, grad_k = _rotate_run(grad_q, grad_k, positions, *ctx.how, 1)
        elif need_q:
            grad_q = _rotate_run(grad_q, None, positions, *ctx.how, 1)[0]
        elif need_k:
            grad_k = _rotate_run(grad_k, None, positions, *ctx.how, 1)[0]
        return grad_q if need_q else None, grad_k if need_k else None, None, None, None, None, None


def _rotate_check(q, k, positions, sections, base):
    _check(q, "q")
    if q.dim() != 4:
        raise ValueError("q must have shape (batch, tokens, heads, head_dim), got %s" % (tuple(q.shape),))
    if k is not None:
        _check(k, "k", q, "q")
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise ValueError("k must have shape (%d, %d, kv_heads, %d), got %s" % (q.shape[0], q.shape[1], q.shape[3], tuple(k.shape)))
    if not torch.is_tensor(positions):
        raise TypeError("positions must be a torch tensor, got %s" % type(positions).__name__)
    _cabi.forward_only("rotate_positions (positions)", positions)
    if positions.dtype not in _POSITION_TYPES:
        raise ValueError("positions must be int32, int64, float32 or float64, got %s" % positions.dtype)
    if tuple(positions.shape) not in (tuple(q.shape[:2]) + (len(sections),), (q.shape[1], len(sections))):
        raise ValueError("positions must have shape %s or %s, got %s" % (tuple(q.shape[:2]) + (len(sections),),
                                                                         (q.shape[1], len(sections)), tuple(positions.shape)))
    _cabi.same_device(q, "q", positions=positions)
    if not (1 <= len(sections) <= 4) or min(sections) < 0 or not 1 <= sum(sections) <= q.shape[3] // 2:
        raise ValueError("sections must list the pairs of 1 to 4 axes, %d in all at most, got %s" % (q.shape[3] // 2, sections))
    if q.shape[2] == 0 or (k is not None and k.shape[2] == 0):
        raise ValueError("q and k must have at least one head")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive and finite, got %r" % (base,))


def _rotate_usual(q, k, positions, sections, base):
    """Whether this is a call with q, k and positions of every sequence in which nothing is wrong."""
    try:
        b, n, heads, dim = q.shape
        kb, kn, k_heads, k_dim = k.shape
        pb, pn, axes = positions.shape
        return (q.is_cuda and q.dtype in _DTYPES and q.dtype == k.dtype and positions.dtype in _POSITION_TYPES
                and not positions.requires_grad and q.get_device() == k.get_device() == positions.get_device()
                and b == kb == pb and n == kn == pn and dim == k_dim and heads > 0 and k_heads > 0 and axes == len(sections)
                and 1 <= axes <= 4 and min(sections) >= 0 and 1 <= sum(sections) <= dim // 2 and 0.0 < base < math.inf)
    except (AttributeError, TypeError, ValueError):
        return False


def rotate_positions(q, k, positions, sections, *, base=10000.0, shared_spectrum=False, pairs=False):
    """Rotary positions with several axes: returns (q, k) with the first 2 * sum(sections) values of every head turned pair by
    pair, the rest copied.  Both come from one launch; k may be None.

    q (batch, tokens, heads, head_dim), k (batch, tokens, kv_heads, head_dim); positions (batch, tokens, axes) or
    (tokens, axes), int32, int64, float32 or float64; sections: the pairs of each axis (1 to 4 axes, at most 128 pairs).  Pair
    i turns by position[axis] * base ** -e, with e its place in the axis' section over the section's pairs or, with
    shared_spectrum, i over all pairs.  Pairs are (i, i + all pairs), or neighbours (2i, 2i + 1) with pairs=True.  Angles are
    float64, so positions of millions keep their place.  Differentiable with respect to q and k."""
    given = tuple(sections)
    sections = tuple(map(int, given))
    if given != sections:
        raise ValueError("sections must be whole numbers of pairs, got %r" % (given,))
    if not _rotate_usual(q, k, positions, sections, base):
        _rotate_check(q, k, positions, sections, base)
    _cabi.no_tangents("rotate_positions", q, k, positions)
    positions = positions.contiguous()
    how = (sections, float(base), int(bool(shared_spectrum)), int(bool(pairs)))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotate.apply(q, k, positions, *how)
    return _rotate_run(q, k, positions, *how, 0)


# ---- attention with a sliding window -----------------------------------------------------------------------------------


def _tokens(t):
    """`t` (batch, tokens, heads, head_dim) as the attention kernels read it: last axis contiguous, base and strides multiples
    of 16 bytes, tokens a head or more and less than 2^25 bytes apart.  Other layouts are copied."""
    aligned = t.data_ptr() % 16 == 0
    if aligned and t.is_contiguous() and t.shape[2] * t.shape[3] < 1 << 22:
        return t
    size = t.element_size()
    vec = 16 // size
    if (aligned and t.stride(3) == 1 and all(st % vec == 0 or n == 1 for st, n in zip(t.stride()[:3], t.shape))
            and (t.shape[1] <= 1 or t.shape[3] <= t.stride(1) < (1 << 25) // size)):
        return t
    c = t.contiguous()
    return c if c.data_ptr() % 16 == 0 else c.clone()


def _window_run(q, k, v, lengths, visible, how, for_backward):
    q, k, v = _tokens(q), _tokens(k), _tokens(v)
    b, n, heads, dim = q.shape
    out = torch.empty((b, n, heads, dim), dtype=q.dtype, device=q.device)
    saved = None
    if for_backward:
        saved = _workspace(_cabi.load().mvx_window_attention_saved_bytes(_DTYPES[q.dtype], b, n, heads, dim), q.device)
    _run(q.get_device(), "window_attention", "mvx_window_attention", q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
         v.data_ptr(), _strides(v), _DTYPES[q.dtype], b, n, heads, k.shape[2], dim, *how, _pointer(lengths), _pointer(visible),
         out.data_ptr(), _pointer(saved))
    return q, k, v, out, saved


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, visible, how):
        q, k, v, out, saved = _window_run(q, k, v, lengths, visible, how, True)
        ctx.save_for_backward(q, k, v, out, saved, lengths, visible)
        ctx.how = how
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, saved, lengths, visible = ctx.saved_tensors
        left, right, sinks, scale = ctx.how
        b, n, heads, dim = q.shape
        kv_heads = k.shape[2]
        grad = _tokens(grad)
        grad_q = torch.empty((b, n, heads, dim), dtype=q.dtype, device=q.device)
        grad_k = torch.empty((b, n, kv_heads, dim), dtype=q.dtype, device=q.device)
        grad_v = torch.empty_like(grad_k)
        ws = _workspace(_cabi.load().mvx_window_attention_backward_workspace_bytes(b, n, heads, kv_heads, dim, left, sinks), q.device)
        _run(q.get_device(), "window_attention", "mvx_window_attention_backward", q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
             v.data_ptr(), _strides(v), out.data_ptr(), saved.data_ptr(), grad.data_ptr(), _strides(grad), _DTYPES[q.dtype], b, n,
             heads, kv_heads, dim, left, right, sinks, scale, _pointer(lengths), _pointer(visible), grad_q.data_ptr(),
             grad_k.data_ptr(), grad_v.data_ptr(), ws.data_ptr(), ws.numel())
        need = ctx.needs_input_grad
        return grad_q if need[0] else None, grad_k if need[1] else None, grad_v if need[2] else None, None, None, None


def _check_dim(dim):
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError("head_dim must be a multiple of 8 up to 128, got %d" % dim)


def _check_scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be positive and finite, got %r" % (scale,))
    return float(scale)


def _check_lengths(lengths, batch, like, like_name):
    if not torch.is_tensor(lengths):
        raise TypeError("lengths must be a torch tensor, got %s" % type(lengths).__name__)
    if lengths.dtype != torch.int64 or lengths.shape != (batch,):
        raise ValueError("lengths must be int64 of shape (%d,), got %s %s" % (batch, lengths.dtype, tuple(lengths.shape)))
    if lengths.get_device() != like.get_device():
        _cabi.same_device(like, like_name, lengths=lengths)


def _check_sinks(sinks):
    if type(sinks) is int and sinks >= 0:
        return sinks
    if sinks != int(sinks) or sinks < 0:
        raise ValueError("sinks must be a whole number, 0 or more, got %r" % (sinks,))
    return int(sinks)


def window_attention(q, k, v, window, sinks=0, *, lengths=None, visible=None, scale=None):
    """Attention over recorded sequences with a sliding window and first tokens that stay visible.

    q (batch, tokens, heads, head_dim), k and v (batch, tokens, kv_heads, head_dim), heads a multiple of kv_heads (head h reads
    key/value head h // (heads // kv_heads)), head_dim a multiple of 8 up to 128; any strides.  window = (left, right): query i
    sees key j if j <= i + right and (j >= i - left or j < sinks); None = no limit on that side; (left, 0) is causal.
    lengths (batch,) int64: tokens of each sequence of a padded batch; visible (batch, tokens) bool: False hides a token (a
    frame without a detection) from every query, itself included.  Values of hidden tokens and of the padding never enter a
    product, whatever they hold; values that are not finite reach the queries that see them and no others.  A query that sees no
    key (or scores of minus infinity alone), and the padding, give zeros and pass no gradient.
    scale: of the scores, head_dim ** -0.5 if None.  Returns (batch, tokens, heads, head_dim).

    Differentiable with respect to q, k and v.  lengths and visible must not be changed between forward and backward."""
    _check_qkv(q, k, v)
    if q.dim() != 4:
        raise ValueError("q must have shape (batch, tokens, heads, head_dim), got %s" % (tuple(q.shape),))
    b, n, heads, dim = q.shape
    _check_dim(dim)
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 4 or t.shape != (b, n, k.shape[2], dim):
            raise ValueError("%s must have shape (%d, %d, kv_heads, %d) with k's heads, got %s" % (name, b, n, dim, tuple(t.shape)))
    if heads == 0 or k.shape[2] == 0 or heads % k.shape[2]:
        raise ValueError("heads (%d) must be a multiple of kv_heads (%d)" % (heads, k.shape[2]))
    left, right = window
    left, right = n if left is None else left, n if right is None else right
    if left != int(left) or right != int(right) or left < 0 or right < 0:
        raise ValueError("window must be two whole numbers, 0 or more, or None, got %r" % (window,))
    if lengths is not None:
        _check_lengths(lengths, b, q, "q")
        lengths = lengths.contiguous()
    if visible is not None:
        if not torch.is_tensor(visible):
            raise TypeError("visible must be a torch tensor, got %s" % type(visible).__name__)
        if visible.dtype != torch.bool or visible.shape != (b, n):
            raise ValueError("visible must be bool of shape (%d, %d), got %s %s" % (b, n, visible.dtype, tuple(visible.shape)))
        if visible.get_device() != q.get_device():
            _cabi.same_device(q, "q", visible=visible)
        visible = visible.contiguous()
    how = (min(int(left), n), min(int(right), n), min(_check_sinks(sinks), n), _check_scale(scale, dim))
    _cabi.no_tangents("window_attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, lengths, visible, how)
    return _window_run(q, k, v, lengths, visible, how, False)[3]


# ---- streams: a ring of cached tokens ----------------------------------------------------------------------------------


def _check_caches(k_cache, v_cache, like, kv_heads, sinks):
    batch, dim = like.shape[0], like.shape[-1]
    try:
        slots = k_cache.shape[1]
        if (k_cache.dtype == v_cache.dtype == like.dtype and like.get_device() == k_cache.get_device() == v_cache.get_device()
                and k_cache.shape == v_cache.shape == (batch, slots, kv_heads, dim) and slots > sinks and k_cache.is_contiguous()
                and v_cache.is_contiguous()):
            k_at, v_at = k_cache.data_ptr(), v_cache.data_ptr()
            if k_at % 16 == 0 and v_at % 16 == 0 and abs(k_at - v_at) >= k_cache.nbytes:
                return
    except (AttributeError, IndexError):
        pass
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check(c, name, like, "k")
        if c.dim() != 4 or c.shape[0] != batch or c.shape[2:] != (kv_heads, dim) or c.shape != k_cache.shape:
            raise ValueError("%s must have shape (%d, sinks + window, %d, %d), both alike, got %s"
                             % (name, batch, kv_heads, dim, tuple(c.shape)))
        if not c.is_contiguous() or c.data_ptr() % 16:
            raise ValueError("%s must be contiguous and 16-byte aligned: it is written in place" % name)
    if k_cache.shape[1] <= sinks:
        raise ValueError("the caches hold %d slots: more than sinks (%d) are needed" % (k_cache.shape[1], sinks))
    if batch:
        raise ValueError("k_cache and v_cache must be two tensors that do not overlap")


def _written(*tensors):
    """Tells autograd that a kernel has written these tensors, as torch's own in-place operations do: a backward that saved
    one of them raises instead of using the new values."""
    torch.autograd.graph.increment_version(tensors)


def window_cache_fill(k, v, k_cache, v_cache, lengths, sinks=0):
    """Fills the rings of window_attention_step, in place, from the first lengths[b] tokens of recorded sequences.

    k, v (batch, tokens, kv_heads, head_dim); k_cache, v_cache (batch, sinks + window, kv_heads, head_dim), contiguous; lengths
    (batch,) int64.  Token t goes to slot t if t < sinks, else to slot sinks + (t - sinks) % window; of each sequence the first
    `sinks` and the last `window` tokens are stored and slots that no token belongs to stay as they are.  The same `lengths`
    (at most `tokens` each) is what the next window_attention_step takes.  Forward only."""
    _check_qkv(k, k, v)
    if k.dim() != 4:
        raise ValueError("k must have shape (batch, tokens, kv_heads, head_dim), got %s" % (tuple(k.shape),))
    if v.shape != k.shape:
        raise ValueError("v must have k's shape %s, got %s" % (tuple(k.shape), tuple(v.shape)))
    b, n, kv_heads, dim = k.shape
    _check_dim(dim)
    sinks = _check_sinks(sinks)
    _check_caches(k_cache, v_cache, k, kv_heads, sinks)
    _check_lengths(lengths, b, k, "k")
    if torch.is_grad_enabled():
        _cabi.forward_only("window_cache_fill", k, v, k_cache, v_cache)
    _cabi.no_tangents("window_cache_fill", k, v, k_cache, v_cache)
    k, v, lengths = _tokens(k), _tokens(v), lengths.contiguous()
    _run(k.get_device(), "window_cache_fill", "mvx_window_cache_fill", k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
         _DTYPES[k.dtype], lengths.data_ptr(), b, n, kv_heads, dim, k_cache.shape[1] - sinks, sinks, k_cache.data_ptr(),
         v_cache.data_ptr())
    _written(k_cache, v_cache)


def window_attention_step(q, k, v, k_cache, v_cache, lengths, sinks=0, *, scale=None):
    """One new token of each stream: stores its k and v in the ring, attends over what the ring holds, and adds 1 to
    `lengths`, all in place and on the device (so a captured call can be replayed frame by frame).

    q (batch, heads, head_dim), k and v (batch, kv_heads, head_dim); k_cache, v_cache (batch, sinks + window, kv_heads,
    head_dim) and lengths (batch,) int64 as window_cache_fill leaves them, or with lengths 0 for streams that begin.  Returns
    (batch, heads, head_dim): the row that window_attention gives the token with window (window - 1, 0).  A negative length
    marks an idle stream: its slots and length stay as they are and its row is zero.  Two calls on the same ring must not
    overlap.  Forward only."""
    _check_qkv(q, k, v)
    if q.dim() != 3:
        raise ValueError("q must have shape (batch, heads, head_dim), got %s" % (tuple(q.shape),))
    b, heads, dim = q.shape
    _check_dim(dim)
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape != (b, k.shape[1], dim):
            raise ValueError("%s must have shape (%d, kv_heads, %d) with k's heads, got %s" % (name, b, dim, tuple(t.shape)))
    kv_heads = k.shape[1]
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("heads (%d) must be a multiple of kv_heads (%d)" % (heads, kv_heads))
    sinks = _check_sinks(sinks)
    _check_caches(k_cache, v_cache, k, kv_heads, sinks)
    _check_lengths(lengths, b, q, "q")
    if not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous: it is written in place")
    if torch.is_grad_enabled():
        _cabi.forward_only("window_attention_step", q, k, v, k_cache, v_cache)
    _cabi.no_tangents("window_attention_step", q, k, v, k_cache, v_cache)
    scale = _check_scale(scale, dim)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    window = k_cache.shape[1] - sinks
    out = torch.empty((b, heads, dim), dtype=q.dtype, device=q.device)
    n_bytes = _cabi.load().mvx_window_attention_step_workspace_bytes(_DTYPES[q.dtype], b, heads, kv_heads, dim, window, sinks)
    ws = _workspace(n_bytes, q.device) if n_bytes else None
    _run(q.get_device(), "window_attention_step", "mvx_window_attention_step", q.data_ptr(), k.data_ptr(), v.data_ptr(),
         _DTYPES[q.dtype], b, heads, kv_heads, dim, window, sinks, scale, k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(),
         out.data_ptr(), _pointer(ws), n_bytes)
    _written(k_cache, v_cache, lengths)
    return out
