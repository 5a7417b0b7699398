"""float64 oracle of the sequence operators (poseestimation_amd.temporal), on the CPU, written from their formulas, with bounds
on what an implementation may be off that forms products and sums in float32 and rounds to the element type where the kernels
say they do (results, softmax weights, score gradients).

Notation of the bounds: u = half a step of the element type (a rounding is off by at most u times the value), e = 2^-24 the same
for float32.  A float32 sum of n products is off by at most n e times the sum of their magnitudes (to first order); constants
are rounded up."""
import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def layer_norm(x, weight, bias, eps, dtype, grad=None):
    """-> (y, bound) or (y, bound, (dx, dw, db), (their bounds)); x (rows, width) etc. already float64."""
    u, width = half_step(dtype), x.shape[-1]
    w = weight if weight is not None else torch.ones(width, dtype=torch.float64)
    b = bias if bias is not None else torch.zeros(width, dtype=torch.float64)
    mean = x.sum(-1, keepdim=True) / width
    c = x - mean
    r = 1.0 / torch.sqrt((c * c).sum(-1, keepdim=True) / width + eps)
    h = c * r
    y = h * w + b
    # sums run over at most 64 terms in a lane, then a tree and the waves: fewer than 96 roundings for any width tested
    n = 96 * E
    size = r * x.abs().sum(-1, keepdim=True) / width  # the mean's error, in units of the row's deviation
    h_err = n * (size + 1) + (n + 8 * E) * h.abs()
    bound = u * y.abs() + w.abs() * h_err + 4 * E * (y.abs() + b.abs())
    if grad is None:
        return y, bound
    a = grad * w
    am, ahm = a.sum(-1, keepdim=True) / width, (a * h).sum(-1, keepdim=True) / width
    dx = r * (a - am - h * ahm)
    dw, db = (grad * h).sum(0), grad.sum(0)
    mag = a.abs().mean(-1, keepdim=True)
    ah_mag = (a * h).abs().mean(-1, keepdim=True)
    dx_err = u * dx.abs() + r * (n * mag + (a.abs() * h_err).mean(-1, keepdim=True) * h.abs() + n * ah_mag * h.abs()
                                 + h_err * ahm.abs() + 16 * E * (a.abs() + am.abs() + (h * ahm).abs()))
    rows = x.shape[0]
    k = (64 + rows) * E  # rows of a workgroup one after the other, then the workgroups
    dw_err = u * dw.abs() + k * (grad * h).abs().sum(0) + (grad.abs() * h_err).sum(0)
    db_err = u * db.abs() + k * grad.abs().sum(0)
    return y, bound, (dx, dw, db), (dx_err, dw_err, db_err)


def rotation_angles(positions, sections, base, shared):
    """(..., tokens, pairs) float64."""
    total, parts, first = sum(sections), [], 0
    for axis, count in enumerate(sections):
        for j in range(count):
            e = (first + j) / total if shared else j / count
            parts.append(positions[..., axis].double() * float(base) ** -e)
        first += count
    return torch.stack(parts, -1)


def rotate(x, positions, sections, base, shared, pairs, dtype, inverse=False):
    """x (batch, tokens, heads, dim) float64 -> (y, bound)."""
    angle = rotation_angles(positions, sections, base, shared)
    if angle.dim() == 2:
        angle = angle[None]
    angle = -angle[:, :, None, :] if inverse else angle[:, :, None, :]
    n = angle.shape[-1]
    at = torch.arange(n)
    one, two = (2 * at, 2 * at + 1) if pairs else (at, at + n)
    c, s = torch.cos(angle), torch.sin(angle)
    y, bound = x.clone(), torch.zeros_like(x)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, a * s + b * c
    # reduced revolutions in float32 (half a step of 1/2: 2 pi 2^-26 radians), cos and sin within 2 steps, two products
    size = (a.abs() + b.abs()) * 8 * E
    u = half_step(dtype)
    bound[..., one], bound[..., two] = size + u * y[..., one].abs(), size + u * y[..., two].abs()
    return y, bound


def seen_pairs(n, left, right, sinks, length, visible):
    """(queries, keys) bool of one sequence."""
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    left, right = n if left is None else left, n if right is None else right
    seen = (j <= i + right) & ((j >= i - left) | (j < sinks))
    if length is not None:
        seen &= (i < length) & (j < length)
    if visible is not None:
        seen &= visible[None, :]
    return seen


def attention(q, k, v, window, sinks, dtype, lengths=None, visible=None, scale=None, grad=None):
    """q (batch, n, heads, dim), k, v (batch, n, kv_heads, dim), float64; hidden values may be anything.
    -> (o, bound) or (o, bound, (dq, dk, dv), (bounds))."""
    b, n, heads, dim = q.shape
    share = heads // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    u = half_step(dtype)
    flat = 2.0 ** -25 if dtype == torch.float16 else 0.0  # float16 values below 2^-14 are rounded to multiples of 2^-24
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    bounds = [torch.zeros_like(t) for t in (q, k, v)]
    for s in range(b):
        length = None if lengths is None else int(lengths[s])
        seen = seen_pairs(n, window[0], window[1], sinks, length, None if visible is None else visible[s])
        some = seen.any(-1, keepdim=True)
        used = seen.any(0)[:, None]
        for h in range(heads):
            kh, vh = (torch.where(used, t[s, :, h // share], 0.0) for t in (k, v))
            qh = torch.where(some, q[s, :, h], 0.0)
            x = torch.where(seen, scale * (qh @ kh.T), -torch.inf)
            top = torch.where(some, x.max(-1, keepdim=True).values, 0.0)
            e = torch.exp(x - top)
            total = e.sum(-1, keepdim=True)
            p = torch.where(some, e / torch.where(some, total, 1.0), 0.0)
            o = p @ vh
            # a weight: its score (dim products, the scaling, the running maximum), exp, the sum of n weights, the division
            x_err = torch.where(seen, scale * (qh.abs() @ kh.abs().T), 0.0) * (dim + 4) * E
            rel = 2 * x_err.max(-1, keepdim=True).values + (n + 64) * E + 4 * E * top.abs()
            pv = p @ vh.abs()
            out[s, :, h] = o
            low = flat * seen.double() @ vh.abs()
            bound[s, :, h] = u * (o.abs() + pv) + (rel + n * E) * pv + low + flat
            if grad is None:
                continue
            g = torch.where(some, grad[s, :, h], 0.0)
            dp = torch.where(seen, g @ vh.T, 0.0)
            delta = (g * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            dp_err = torch.where(seen, g.abs() @ vh.abs().T, 0.0) * (dim + 4) * E
            delta_err = (g.abs() * (bound[s, :, h] + (dim + 4) * E * o.abs())).sum(-1, keepdim=True)
            ds_err = u * ds.abs() + p * (dp_err + delta_err) + (rel + 8 * E) * p * (dp.abs() + delta.abs())
            ds_err = ds_err + torch.where(seen, flat, 0.0)
            p_err = (u + rel) * p + torch.where(seen, flat, 0.0)
            grads[0][s, :, h] = scale * ds @ kh
            bounds[0][s, :, h] = scale * (ds_err + n * E * ds.abs()) @ kh.abs()
            grads[1][s, :, h // share] += scale * ds.T @ qh
            bounds[1][s, :, h // share] += scale * (ds_err + n * share * E * ds.abs()).T @ qh.abs()
            grads[2][s, :, h // share] += p.T @ g
            bounds[2][s, :, h // share] += (p_err + n * share * E * p).T @ g.abs()
    if grad is None:
        return out, bound
    for g, e in zip(grads, bounds):
        e += u * g.abs() + flat
    return out, bound, tuple(grads), tuple(bounds)


def cache_slot(token, sinks, window):
    return token if token < sinks else sinks + (token - sinks) % window


def fill(k, caches, lengths, sinks):
    """Stores the tokens a ring holds of k (batch, n, heads, dim) into `caches`, in place, token after token."""
    window = caches.shape[1] - sinks
    for s in range(k.shape[0]):
        for t in range(min(int(lengths[s]), k.shape[1])):
            caches[s, cache_slot(t, sinks, window)] = k[s, t]
