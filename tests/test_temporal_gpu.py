"""The sequence operators (poseestimation_amd.temporal) against the float64 oracle, which also gives the bound every element has
to keep (see oracle/temporal_oracle.py for its derivation)."""
import itertools

import pytest
import torch
import torch.autograd.forward_ad as fwd

import temporal_oracle as orc
from poseestimation_amd import _cabi, temporal

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, shape, dtype, leaf=False, spread=1.0, offset=0.0):
    return (torch.randn(shape, generator=g) * spread + offset).to(dtype).to(DEV).requires_grad_(leaf)


def f64(t):
    return t.detach().cpu().double() if t is not None else None


def within(got, want, bound, what):
    got = f64(got)
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), "%s: not finite" % what
    over = (got - want).abs() - bound
    assert (over <= 0).all(), "%s: off by %g where %g is allowed" % (
        what, (got - want).abs().flatten()[over.argmax()], bound.flatten()[over.argmax()])


# ---- layer norm --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 7), (2, 8), (17, 9), (1, 33), (17, 256), (33, 257), (5, 511), (70, 1000),
                                        (300, 1024), (9, 1025), (40, 2047), (600, 2048), (3, 2049), (11, 4097), (2, 8191),
                                        (4, 8192), (3, 16383), (2, 16385), (2, 20000)])
def test_layer_norm(dtype, rows, width):
    g = gen(rows * 100003 + width)
    x = normal(g, (rows, width), dtype, True, 2.0, 0.5)
    w, b = normal(g, (width,), dtype, True, 0.3, 1.0), normal(g, (width,), dtype, True, 0.3)
    up = normal(g, (rows, width), dtype)
    y = temporal.layer_norm(x, w, b, 1e-5)
    assert y.dtype == dtype and y.shape == x.shape
    assert torch.equal(y, temporal.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5))
    got = torch.autograd.grad(y, (x, w, b), up)
    want, bound, grads, bounds = orc.layer_norm(f64(x), f64(w), f64(b), 1e-5, dtype, f64(up))
    within(y, want, bound, "y")
    for name, a, c, e in zip(("dx", "dweight", "dbias"), got, grads, bounds):
        within(a, c, e, name)


@pytest.mark.parametrize("which", ["none", "weight", "bias", "float32", "x only", "parameters only"])
def test_layer_norm_parameters(which):
    g = gen(5)
    dtype = torch.bfloat16
    pdtype = torch.float32 if which == "float32" else dtype
    x = normal(g, (3, 5, 264), dtype, which != "parameters only")
    w = normal(g, (264,), pdtype, which != "x only", 0.3, 1.0) if which not in ("none", "bias") else None
    b = normal(g, (264,), pdtype, which != "x only", 0.3) if which not in ("none", "weight") else None
    up = normal(g, (3, 5, 264), dtype)
    y = temporal.layer_norm(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None and t.requires_grad]
    got = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, up)))
    want, bound, grads, bounds = orc.layer_norm(f64(x).reshape(15, 264), f64(w), f64(b), 1e-5, dtype, f64(up).reshape(15, 264))
    within(y.reshape(15, 264), want, bound, "y")
    for name, t, a, e in zip(("dx", "dw", "db"), (x, w, b), grads, bounds):
        if t is not None and id(t) in got:
            assert got[id(t)].dtype == t.dtype
            within(got[id(t)].reshape(a.shape), a, e, name)


def test_layer_norm_offset_rows_empty_rows_and_strides():
    g = gen(6)
    x = normal(g, (9, 300), torch.float32, spread=1e-3, offset=100.0)  # the variance must not drown in the mean
    within(temporal.layer_norm(x), *orc.layer_norm(f64(x), None, None, 1e-5, torch.float32), "offset rows")
    assert (temporal.layer_norm(torch.full((2, 64), 3.0, device=DEV)) == 0).all()  # a constant row
    e = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = temporal.layer_norm(e, w)
    assert y.shape == (0, 64)
    ge, gw = torch.autograd.grad(y, (e, w), torch.empty_like(y))
    assert ge.shape == (0, 64) and (gw == 0).all()
    base = normal(g, (40, 12, 130), torch.float16)
    t = base.transpose(0, 1)[:, 3:, 1:]  # strides, and a base that is not 16-byte aligned
    want, bound = orc.layer_norm(f64(t).reshape(-1, 129), None, None, 1e-5, torch.float16)
    within(temporal.layer_norm(t).reshape(-1, 129), want, bound, "strided")
    flat = base.flatten()[1:1 + 64 * 129].view(64, 129)
    want, bound = orc.layer_norm(f64(flat), None, None, 1e-5, torch.float16)
    within(temporal.layer_norm(flat), want, bound, "misaligned base")


# ---- rotary positions --------------------------------------------------------------------------------------------------

ROTARY = [
    # batch, tokens, heads, kv_heads, dim, sections, pairs, shared, position type, per sequence
    (1, 1, 1, 1, 8, (4,), False, False, torch.int64, True),
    (1, 17, 8, 8, 64, (8, 12, 12), True, False, torch.int32, True),
    (2, 50, 4, 2, 64, (10, 11, 11), False, True, torch.int32, False),
    (3, 37, 3, 1, 96, (7, 3, 5), False, False, torch.float32, True),
    (2, 29, 2, 2, 80, (1, 1, 1, 2), True, True, torch.float64, True),
    (1, 1200, 4, 4, 128, (16, 24, 24), False, False, torch.int64, True),
    (1, 5, 2, 1, 256, (64, 64), True, False, torch.int32, True),
    (2, 9, 1, 1, 13, (0, 6), False, False, torch.int32, True),
    (1, 11, 5, 5, 40, (3, 2), True, False, torch.int32, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROTARY)
def test_rotate_positions(dtype, case):
    b, n, h, hk, d, sections, pairs, shared, ptype, per_seq = case
    g = gen(n * d)
    q, k = normal(g, (b, n, h, d), dtype, True), normal(g, (b, n, hk, d), dtype, True)
    gq, gk = normal(g, (b, n, h, d), dtype), normal(g, (b, n, hk, d), dtype)
    pos = torch.randint(0, 200000, ((b,) if per_seq else ()) + (n, len(sections)), generator=g).to(ptype)
    if ptype.is_floating_point:
        pos = pos / 64 - 1000  # positions of a voxel grid: fractions, negative ones
    how = dict(base=500.0, shared_spectrum=shared, pairs=pairs)
    qo, ko = temporal.rotate_positions(q, k, pos.to(DEV), sections, **how)
    for got, x in ((qo, q), (ko, k)):
        assert got.dtype == dtype
        within(got, *orc.rotate(f64(x), pos, sections, 500.0, shared, pairs, dtype), "rotated")
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    for got, x in ((dq, gq), (dk, gk)):
        within(got, *orc.rotate(f64(x), pos, sections, 500.0, shared, pairs, dtype, inverse=True), "gradient")
    alone, none = temporal.rotate_positions(q.detach(), None, pos.to(DEV), sections, **how)
    assert none is None and torch.equal(alone, qo)


def test_rotate_positions_far_strided_and_partial_gradients():
    g = gen(3)
    pos = torch.tensor([[0, 0, 0], [2 ** 31 - 1, 5, -7], [10 ** 9 + 1, 123456789, 3], [2 ** 24 + 1, 2 ** 24 + 2, 2 ** 24 + 3]])
    packed = normal(g, (2, 4, 3, 6, 48), torch.float32)
    q, k = packed[:, :, 0], packed[:, :, 1, ::2]
    qo, ko = temporal.rotate_positions(q, k, pos.to(DEV), (8, 8, 8))
    for got, x in ((qo, q), (ko, k)):
        # an angle of 2^31 radians keeps 2^-53 of itself in float64: 5e-7 of a radian in the oracle and in the kernel each
        want, bound = orc.rotate(f64(x), pos, (8, 8, 8), 10000.0, False, False, torch.float32)
        within(got, want, bound + 1e-6 * f64(x).abs().amax(-1, keepdim=True) * 2, "far")
    ql = q.detach().clone().requires_grad_(True)
    qo, ko = temporal.rotate_positions(ql, k, pos.to(DEV), (8, 8, 8))
    dq, = torch.autograd.grad(qo.sum() + ko.sum(), ql)
    want, bound = orc.rotate(torch.ones(2, 4, 6, 48, dtype=torch.float64), pos, (8, 8, 8), 10000.0, False, False, torch.float32, True)
    within(dq, want, bound + 4e-6, "gradient of q alone")
    assert temporal.rotate_positions(q[:, :0], None, pos[:0].to(DEV), (8, 8, 8))[0].shape == (2, 0, 6, 48)
    # values behind the pairs are copied bit for bit, infinities and NaN among them
    x = normal(g, (1, 4, 2, 40), torch.bfloat16)
    x[..., 30:] = float("inf")
    x[..., 35:] = float("nan")
    y, _ = temporal.rotate_positions(x, None, pos.to(DEV), (5, 5, 5))
    assert torch.equal(y[..., 30:].view(torch.int16), x[..., 30:].view(torch.int16)) and torch.isfinite(y[..., :30]).all()


# ---- attention over sequences ------------------------------------------------------------------------------------------

ATTENTION = [
    # batch, tokens, heads, kv_heads, dim, window, sinks, lengths, hidden
    (1, 1, 1, 1, 8, (0, 0), 0, None, False),
    (2, 3, 2, 1, 16, (1, 0), 1, (0, 3), False),
    (1, 63, 2, 2, 32, (None, 0), 0, None, False),
    (1, 64, 1, 1, 64, (None, None), 0, None, True),
    (2, 65, 4, 2, 64, (7, 7), 3, (65, 1), True),
    (1, 200, 2, 1, 40, (0, 0), 0, None, True),
    (1, 257, 4, 4, 64, (16, 16), 0, None, True),
    (2, 300, 6, 2, 96, (33, 5), 70, (300, 129), False),
    (1, 500, 2, 1, 128, (40, 0), 4, None, False),
    (1, 700, 2, 2, 72, (64, 0), 130, (650,), True),
    (2, 900, 2, 1, 32, (20, 3), 2, (900, 641), True),
    (1, 1300, 1, 1, 64, (None, 0), 5, None, False),
]


def attention_case(case, dtype, seed=0, leaf=False):
    b, n, h, hk, d, window, sinks, lengths, hidden = case
    g = gen(n * 31 + d + seed)
    q, k, v = (normal(g, (b, n, heads, d), dtype, leaf) for heads in (h, hk, hk))
    up = normal(g, (b, n, h, d), dtype)
    lengths = torch.tensor(lengths, dtype=torch.int64) if lengths is not None else None
    visible = torch.rand((b, n), generator=g) < 0.7 if hidden else None
    return q, k, v, up, lengths, visible


def on_gpu(t):
    return t.to(DEV) if t is not None else None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ATTENTION)
def test_window_attention(dtype, case):
    q, k, v, up, lengths, visible = attention_case(case, dtype, leaf=True)
    how = dict(lengths=on_gpu(lengths), visible=on_gpu(visible))
    out = temporal.window_attention(q, k, v, case[5], case[6], **how)
    assert out.dtype == dtype and out.shape == q.shape
    assert torch.equal(out, temporal.window_attention(q.detach(), k.detach(), v.detach(), case[5], case[6], **how))
    got = torch.autograd.grad(out, (q, k, v), up, retain_graph=True)
    want, bound, grads, bounds = orc.attention(f64(q), f64(k), f64(v), case[5], case[6], dtype, lengths, visible, grad=f64(up))
    within(out, want, bound, "out")
    for name, a, c, e in zip(("dq", "dk", "dv"), got, grads, bounds):
        within(a, c, e, name)
    for a, c in zip(got, torch.autograd.grad(out, (q, k, v), up)):  # sums in a fixed order
        assert torch.equal(a, c)


def test_window_attention_strides_and_broadcast_inputs():
    b, n, h, hk, d = 2, 130, 4, 2, 48
    g = gen(11)
    for dtype in DTYPES:
        # q, k, v as slices of one packed projection; k and v then expanded over the batch
        packed = normal(g, (b, n, h + 2 * hk, d), dtype, True)
        up = normal(g, (b, n, h, d), dtype)
        q, k, v = packed.split((h, hk, hk), dim=2)
        out = temporal.window_attention(q, k, v, (20, 4), 1)
        got, = torch.autograd.grad(out, packed, up.transpose(1, 2).contiguous().transpose(1, 2))  # a strided gradient too
        want, bound, grads, bounds = orc.attention(f64(q), f64(k), f64(v), (20, 4), 1, dtype, grad=f64(up))
        within(out, want, bound, "packed")
        within(got, torch.cat(grads, 2), torch.cat(bounds, 2), "packed gradient")
        shared = normal(g, (1, n, hk, d), dtype, True)
        ql = normal(g, (b, n, h, d), dtype)
        out = temporal.window_attention(ql, shared.expand(b, n, hk, d), v, (20, 4), 1)
        got, = torch.autograd.grad(out, shared, up)
        want, bound, grads, bounds = orc.attention(f64(ql), f64(shared).expand(b, n, hk, d), f64(v), (20, 4), 1, dtype, grad=f64(up))
        within(out, want, bound, "broadcast keys")
        total = grads[1].sum(0, keepdim=True)
        step = orc.half_step(dtype)
        within(got, total, bounds[1].sum(0, keepdim=True) + step * grads[1].abs().sum(0, keepdim=True) + step * total.abs(), "their gradient")
        # layouts that have to be copied: heads before tokens, an odd offset, reversed strides of the last axis
        odd = normal(g, (b, n, h, d + 1), dtype)[..., 1:]
        last = normal(g, (b, n, d, hk), dtype).transpose(2, 3)
        want, bound = orc.attention(f64(odd), f64(last), f64(last), (20, 4), 1, dtype)
        within(temporal.window_attention(odd, last, last, (20, 4), 1), want, bound, "copied layouts")


@pytest.mark.parametrize("dtype", DTYPES)
def test_window_attention_hidden_values_are_never_read_into_a_product(dtype):
    case = (2, 190, 2, 1, 64, (30, 10), 3, (190, 140), True)
    q, k, v, up, lengths, visible = attention_case(case, dtype)
    visible[1, :3] = False  # hidden sinks
    clean = [t.clone() for t in (q, k, v, up)]
    how = dict(lengths=on_gpu(lengths), visible=on_gpu(visible))

    def both(q, k, v, up):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = temporal.window_attention(*leaves, case[5], case[6], **how)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]

    want = both(*clean)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        k[~visible.to(DEV)], v[~visible.to(DEV)] = bad, bad
        for t in (q, k, v, up):
            t[1, 140:] = bad
        for a, c in zip(both(q, k, v, up), want):
            assert torch.equal(a, c)
    assert all((t[1, 140:] == 0).all() for t in want)
    hidden = ~visible.to(DEV)
    assert (want[2][hidden] == 0).all() and (want[3][hidden] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_window_attention_values_that_are_not_finite_reach_those_that_see_them_alone(dtype):
    n, window, sinks, d = 400, (40, 9), 2, 32
    g = gen(21)
    q, k, v, up = (normal(g, (1, n, heads, d), dtype) for heads in (2, 1, 1, 2))

    def both(q, k, v):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = temporal.window_attention(*leaves, window, sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]

    seen = orc.seen_pairs(n, *window, sinks, None, None)
    clean = both(q, k, v)
    want, bound, grads, bounds = orc.attention(f64(q), f64(k), f64(v), window, sinks, dtype, grad=f64(up))
    for j, poisoned in ((150, v), (150, k), (1, v)):
        keep = poisoned.clone()
        poisoned[0, j] = float("nan")
        out, dq, dk, dv = both(q, k, v)
        poisoned.copy_(keep)
        hit = seen[:, j]  # queries that see the token
        assert torch.isnan(out[0, hit]).all()
        clear = ~hit
        within(out[0, clear], want[0, clear], bound[0, clear], "queries that do not see it")
        within(dq[0, clear], grads[0][0, clear], bounds[0][0, clear], "their gradient")
        beyond = ~(seen[hit].any(0))  # keys that no such query sees
        if beyond.any():
            within(dk[0, beyond], grads[1][0, beyond], bounds[1][0, beyond], "keys that share no query with it")
            within(dv[0, beyond], grads[2][0, beyond], bounds[2][0, beyond], "their values")
    assert all(torch.equal(a, c) for a, c in zip(both(q, k, v), clean))


def test_window_attention_empty_and_extreme():
    for shape in ((0, 5, 2, 16), (2, 0, 2, 16)):
        t = torch.empty(shape, device=DEV, requires_grad=True)
        out = temporal.window_attention(t, t, t, (1, 1))
        assert out.shape == shape
        assert torch.autograd.grad(out.sum(), t)[0].shape == shape
    g = gen(4)
    q, k, v = (normal(g, (1, 70, 1, 16), torch.float32) for _ in range(3))
    nobody = torch.zeros(1, 70, dtype=torch.bool, device=DEV)
    assert (temporal.window_attention(q, k, v, (None, None), visible=nobody) == 0).all()
    assert (temporal.window_attention(q, k, v, (None, None), lengths=torch.tensor([-5], device=DEV)) == 0).all()
    every = temporal.window_attention(q, k, v, (None, None))
    assert torch.equal(every, temporal.window_attention(q, k, v, (10 ** 12, 10 ** 12), 10 ** 12, lengths=torch.tensor([10 ** 12], device=DEV)))
    # scores of thousands: the largest one takes all
    out = temporal.window_attention(q * 1000, k * 1000, v, (None, None))
    top = (f64(q)[0, :, 0] @ f64(k)[0, :, 0].T).argmax(-1)
    # every other weight is 0 and the top one some w near 1 (the exponent of 2 is score * scale less the rounded maximum), so
    # the row is fl(fl(w v) * fl(1 / w)): three roundings of 2^-24 each, (1 + 2^-24)^3 - 1 < 3.0001 * 2^-24
    want = v[0, :, 0].cpu()[top]
    assert ((out[0, :, 0].cpu() - want).abs() <= 3.0001 * 2.0 ** -24 * want.abs()).all()
    scaled = temporal.window_attention(q, k, v, (5, 5), scale=0.7)
    within(scaled, *orc.attention(f64(q), f64(k), f64(v), (5, 5), 0, torch.float32, scale=0.7), "scale")


# ---- streams -----------------------------------------------------------------------------------------------------------


def step_oracle(q, kc, vc, lengths, sinks, dtype, scale=None):
    """One step over the float64 rings kc, vc in which the new token has been stored; lengths before the step."""
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s in range(q.shape[0]):
        length = int(lengths[s])
        if length < 0:
            continue
        held = min(length + 1, kc.shape[1])
        # the same softmax as a query that sees `held` keys
        n = held
        qs = torch.zeros(1, n, q.shape[1], q.shape[2], dtype=torch.float64)
        qs[0, -1] = q[s]
        o, e = orc.attention(qs, kc[s:s + 1, :n], vc[s:s + 1, :n], (None, None), 0, dtype, scale=scale)
        out[s], bound[s] = o[0, -1], e[0, -1]
    return out, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,window,sinks", [(1, 1, 8, 1, 0), (2, 2, 32, 5, 2), (4, 2, 64, 64, 4), (8, 2, 40, 70, 0),
                                                            (6, 1, 96, 33, 1), (16, 1, 128, 300, 16), (3, 3, 72, 1000, 70)])
def test_window_attention_step(dtype, heads, kv_heads, dim, window, sinks):
    g = gen(window * dim + heads)
    cap = sinks + window
    b = 5
    kc, vc = normal(g, (b, cap, kv_heads, dim), dtype), normal(g, (b, cap, kv_heads, dim), dtype)
    lengths = torch.tensor([0, max(0, cap - 2), -1, 3 * cap + 1, max(0, sinks - 1)], dtype=torch.int64)
    kc[0], vc[0] = float("nan"), float("nan")  # a ring that holds nothing yet is not read
    dl = lengths.to(DEV)
    for _ in range(4):
        q = normal(g, (b, heads, dim), dtype)
        k, v = normal(g, (b, kv_heads, dim), dtype), normal(g, (b, kv_heads, dim), dtype)
        want_k, want_v = f64(kc), f64(vc)
        for s in range(b):
            if lengths[s] >= 0:
                at = orc.cache_slot(int(lengths[s]), sinks, window)
                want_k[s, at], want_v[s, at] = f64(k)[s], f64(v)[s]
        out = temporal.window_attention_step(q, k, v, kc, vc, dl, sinks)
        assert torch.equal(f64(kc).nan_to_num(9.0), want_k.nan_to_num(9.0)) and torch.equal(f64(vc).nan_to_num(9.0), want_v.nan_to_num(9.0))
        want, bound = step_oracle(f64(q), want_k, want_v, lengths, sinks, dtype)
        within(out, want, bound, "step")
        assert (out[2] == 0).all()
        lengths = torch.where(lengths >= 0, lengths + 1, lengths)
        assert torch.equal(dl.cpu(), lengths)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,window,sinks,dim", [(1, 4, 0, 8), (50, 7, 3, 40), (64, 100, 4, 64), (333, 64, 70, 128), (9, 3, 20, 16)])
def test_window_cache_fill(dtype, n, window, sinks, dim):
    g = gen(n)
    hk, b = 3, 4
    packed = normal(g, (b, n, 2 * hk, dim), dtype)
    k, v = packed.split((hk, hk), dim=2)
    kc, vc = normal(g, (b, sinks + window, hk, dim), dtype), normal(g, (b, sinks + window, hk, dim), dtype)
    lengths = torch.tensor([n, 0, max(1, n // 2), -1])
    want_k, want_v = f64(kc), f64(vc)
    orc.fill(f64(k), want_k, lengths, sinks)
    orc.fill(f64(v), want_v, lengths, sinks)
    temporal.window_cache_fill(k, v, kc, vc, lengths.to(DEV), sinks)
    assert torch.equal(f64(kc), want_k) and torch.equal(f64(vc), want_v)
    temporal.window_cache_fill(k, v, kc, vc, (lengths + 10 * n).to(DEV), sinks)  # above n: taken as n
    orc.fill(f64(k), want_k, lengths + 10 * n, sinks)
    assert torch.equal(f64(kc), want_k)


# ---- together ----------------------------------------------------------------------------------------------------------


def block(x, p, positions, attend):
    """One block of a sequence model without its feed-forward part: norm -> projection -> rotate -> attend -> projection."""
    h = temporal.layer_norm(x, p["w"], p["b"])
    q, k, v = (h @ p["in"]).unflatten(-1, (8, 16)).split((4, 2, 2), dim=-2)
    q, k = temporal.rotate_positions(q, k, positions, (4, 2, 2))
    return x + attend(q, k, v).flatten(-2) @ p["out"]


def parameters(g, leaf):
    return {name: normal(g, shape, torch.float32, leaf, spread, offset) for name, shape, spread, offset in
            (("w", (64,), 0.2, 1.0), ("b", (64,), 0.2, 0.0), ("in", (64, 128), 0.12, 0.0), ("out", (64, 64), 0.12, 0.0))}


def oracle_block(x, p, positions, window, sinks, lengths):
    def rotate(t):
        angle = orc.rotation_angles(positions, (4, 2, 2), 10000.0, False)[None, :, None, :]
        a, b = t[..., :8], t[..., 8:]
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    c = x - x.mean(-1, keepdim=True)
    h = c / ((c * c).mean(-1, keepdim=True) + 1e-5).sqrt() * p["w"] + p["b"]
    q, k, v = (h @ p["in"]).unflatten(-1, (8, 16)).split((4, 2, 2), dim=-2)
    q, k, v = rotate(q), rotate(k).repeat_interleave(2, 2), v.repeat_interleave(2, 2)
    seen = torch.stack([orc.seen_pairs(x.shape[1], *window, sinks, int(n), None) for n in lengths])[:, None]
    s = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1) / 4).masked_fill(~seen, -torch.inf)
    a = torch.where(seen.any(-1, keepdim=True), torch.softmax(s.masked_fill(~seen.any(-1, keepdim=True), 0.0), -1), 0.0)
    return x + (a @ v.transpose(1, 2)).transpose(1, 2).flatten(-2) @ p["out"]


def test_a_block_trains_and_streams():
    g = gen(77)
    n, window, sinks = 150, 40, 2
    x, p = normal(g, (2, n, 64), torch.float32, True), parameters(g, True)
    positions = torch.stack((torch.arange(n), torch.arange(n) % 17, torch.arange(n) % 5), -1)
    lengths = torch.tensor([150, 90])
    up = normal(g, (2, n, 64), torch.float32)
    dl = lengths.to(DEV)
    leaves = [x, *p.values()]

    def forward(x, p):
        return block(x, p, positions.to(DEV), lambda q, k, v: temporal.window_attention(q, k, v, (window - 1, 0), sinks, lengths=dl))

    out = forward(x, p)
    got = torch.autograd.grad(out, leaves, up)
    x64 = f64(x).requires_grad_(True)
    p64 = {c: f64(t).requires_grad_(True) for c, t in p.items()}
    want = oracle_block(x64, p64, positions, (window - 1, 0), sinks, lengths)
    assert (f64(out) - want).abs().max() < 1e-5 * want.abs().max()
    # float32 through two products of 64 and 128 terms and 150 keys: relative errors of about sqrt(terms) 2^-24 each
    for a, c in zip(got, torch.autograd.grad(want, [x64, *p64.values()], f64(up))):
        assert (f64(a) - c).abs().max() < 2e-5 * c.abs().max()

    # the same block on a stream: a prompt of 100 and 60 tokens fills the ring, the rest comes one token at a time
    with torch.no_grad():
        start = torch.tensor([100, 60])
        kc, vc = torch.zeros(2, sinks + window, 2, 16, device=DEV), torch.zeros(2, sinks + window, 2, 16, device=DEV)
        state = start.to(DEV)
        pd = {c: t.detach() for c, t in p.items()}

        def prompt(q, k, v):
            temporal.window_cache_fill(k, v, kc, vc, state, sinks)
            return temporal.window_attention(q, k, v, (window - 1, 0), sinks, lengths=state)

        first = block(x, pd, positions.to(DEV), prompt)
        for s in range(2):
            assert (first[s, :start[s]] - out[s, :start[s]]).abs().max() < 1e-5
        for t in range(30):
            now = torch.stack([x[s, start[s] + t] for s in range(2)])[:, None]
            where = torch.stack([positions[start[s] + t] for s in range(2)])[:, None].to(DEV)
            y = block(now, pd, where, lambda q, k, v: temporal.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, state, sinks)[:, None])
            for s in range(2):
                assert (y[s, 0] - out[s, start[s] + t]).abs().max() < 1e-5
        assert torch.equal(state.cpu(), start + 30)


def test_step_under_graph_capture():
    """A captured step is replayed frame by frame: the ring and the lengths advance on the device."""
    g = gen(31)
    b, h, hk, d, window, sinks = 3, 4, 2, 64, 200, 4
    frames = [tuple(normal(g, (b, heads, d), torch.bfloat16) for heads in (h, hk, hk)) for _ in range(6)]
    kc, vc = normal(g, (b, window + sinks, hk, d), torch.bfloat16), normal(g, (b, window + sinks, hk, d), torch.bfloat16)
    lengths = torch.tensor([0, 500, -1], device=DEV)
    eager = [kc.clone(), vc.clone(), lengths.clone()]
    want = [temporal.window_attention_step(*f, *eager, sinks) for f in frames]
    q, k, v = (t.clone() for t in frames[0])
    scratch = [kc.clone(), vc.clone(), lengths.clone()]
    temporal.window_attention_step(q, k, v, *scratch, sinks)  # warm-up outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = temporal.window_attention_step(q, k, v, kc, vc, lengths, sinks)
    for f, w in zip(frames, want):
        for a, c in zip((q, k, v), f):
            a.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        torch.full((1000,), 3.0, device=DEV).sum().item()  # eager work between the replays
    assert torch.equal(kc, eager[0]) and torch.equal(vc, eager[1]) and torch.equal(lengths, eager[2])


def test_training_under_graph_capture_and_on_another_stream():
    g = gen(32)
    n = 300
    x = normal(g, (2, n, 128), torch.bfloat16, True)
    w, c = normal(g, (128,), torch.bfloat16, True, 0.2, 1.0), normal(g, (128,), torch.bfloat16, True, 0.2)
    up = normal(g, (2, n, 4, 16), torch.bfloat16)
    positions = torch.stack((torch.arange(n), torch.arange(n) % 17, torch.arange(n) % 5), -1).to(DEV)
    lengths = torch.tensor([300, 171], device=DEV)

    def step():
        q, k, v = temporal.layer_norm(x, w, c).unflatten(-1, (8, 16)).split((4, 2, 2), dim=-2)
        q, k = temporal.rotate_positions(q, k, positions, (4, 2, 2))
        out = temporal.window_attention(q, k, v, (30, 30), 2, lengths=lengths)
        return [out.detach(), *torch.autograd.grad(out, [x, w, c], up)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        for _ in range(2):
            step()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for k in range(3):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), k
        step()  # eager work between the replays


def test_lengths_changed_between_forward_and_backward_are_refused():
    g = gen(8)
    q, k, v = (normal(g, (1, 20, 1, 16), torch.float32, True) for _ in range(3))
    lengths = torch.tensor([12], device=DEV)
    out = temporal.window_attention(q, k, v, (5, 0), lengths=lengths)
    cache = torch.zeros(2, 1, 6, 1, 16, device=DEV)
    temporal.window_attention_step(q[:, 0].detach(), k[:, 0].detach(), v[:, 0].detach(), cache[0], cache[1], lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals_on_the_gpu():
    t = torch.zeros(2, 10, 4, 16, device=DEV)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        temporal.window_attention(t, t[:, :, :3], t[:, :, :3], (1, 1))
    with pytest.raises(ValueError, match="k is torch.float16"):
        temporal.window_attention(t, t.half(), t, (1, 1))
    with pytest.raises(ValueError, match="multiple of 8"):
        temporal.window_attention(t[..., :12], t[..., :12], t[..., :12], (1, 1))
    with pytest.raises(ValueError, match="window"):
        temporal.window_attention(t, t, t, (-1, 1))
    with pytest.raises(ValueError, match="sinks"):
        temporal.window_attention(t, t, t, (1, 1), -2)
    with pytest.raises(ValueError, match="scale"):
        temporal.window_attention(t, t, t, (1, 1), scale=0.0)
    with pytest.raises(ValueError, match="lengths"):
        temporal.window_attention(t, t, t, (1, 1), lengths=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="visible"):
        temporal.window_attention(t, t, t, (1, 1), visible=torch.zeros(2, 9, dtype=torch.bool, device=DEV))
    with pytest.raises(_cabi.MvxError, match="same device"):
        temporal.window_attention(t, t, t, (1, 1), lengths=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="sections"):
        temporal.rotate_positions(t, None, torch.zeros(10, 2, dtype=torch.int32, device=DEV), (8, 1))
    with pytest.raises(ValueError, match="positions"):
        temporal.rotate_positions(t, None, torch.zeros(10, 3, dtype=torch.int32, device=DEV), (4, 4))
    with pytest.raises(_cabi.MvxError, match="forward-only"):
        temporal.rotate_positions(t, None, torch.zeros(10, 2, device=DEV, requires_grad=True), (4, 4))
    with pytest.raises(ValueError, match="weight"):
        temporal.layer_norm(t, torch.ones(15, device=DEV))
    with pytest.raises(ValueError, match="float32"):
        temporal.layer_norm(t, torch.ones(16, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError, match="eps"):
        temporal.layer_norm(t, eps=float("nan"))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        temporal.layer_norm(t.double())
    q, kv = t[:, 0], t[:, 0, :2]
    cache, n = torch.zeros(2, 5, 2, 16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="two tensors"):
        temporal.window_attention_step(q, kv, kv, cache, cache, n)
    with pytest.raises(ValueError, match="sinks"):
        temporal.window_attention_step(q, kv, kv, cache, cache.clone(), n, 5)
    with pytest.raises(ValueError, match="contiguous"):
        temporal.window_attention_step(q, kv, kv, cache.transpose(0, 1).contiguous().transpose(0, 1), cache.clone(), n)
    with pytest.raises(ValueError, match="lengths"):
        temporal.window_attention_step(q, kv, kv, cache, cache.clone(), n.int())
    with pytest.raises(_cabi.MvxError, match="forward-only"):
        temporal.window_attention_step(q.clone().requires_grad_(True), kv, kv, cache, cache.clone(), n)
    with pytest.raises(ValueError, match="v_cache"):
        temporal.window_cache_fill(t, t, torch.zeros(2, 5, 4, 16, device=DEV), torch.zeros(2, 6, 4, 16, device=DEV), n)
    with pytest.raises(ValueError, match="k_cache"):
        temporal.window_cache_fill(t, t, cache, cache.clone(), n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks,hidden", [((0, 0), 0, False), ((0, 0), 0, True), ((3, 0), 1, True), ((0, 0), 2, False)])
def test_a_query_that_sees_one_key_gives_q_and_k_no_gradient(dtype, window, sinks, hidden):
    """Its weight is 1 whatever the score; what rounding leaves of dp - delta must not pass for a gradient."""
    n = 420
    g = gen(51)
    q, k, v = (normal(g, (2, n, heads, 32), dtype, True) for heads in (4, 2, 2))
    up = normal(g, (2, n, 4, 32), dtype)
    visible = torch.rand((2, n), generator=g) < 0.25 if hidden else None
    lengths = torch.tensor([n, 333])
    out = temporal.window_attention(q, k, v, window, sinks, lengths=on_gpu(lengths), visible=on_gpu(visible))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), up)
    want, bound, grads, bounds = orc.attention(f64(q), f64(k), f64(v), window, sinks, dtype, lengths, visible, grad=f64(up))
    for name, a, c, e in zip(("dq", "dk", "dv"), (dq, dk, dv), grads, bounds):
        within(a, c, e, name)
    for s in range(2):
        seen = orc.seen_pairs(n, *window, sinks, int(lengths[s]), None if visible is None else visible[s])
        alone = seen.sum(-1) == 1
        assert alone.any() and (dq[s, alone] == 0).all()
        only_theirs = ~seen[seen.sum(-1) > 1].any(0)  # keys that no query with a choice sees
        assert (dk[s, only_theirs] == 0).all()


def test_a_query_whose_only_key_is_not_finite_does_not_hide_it():
    q, k, v = (normal(gen(52), (1, 40, 2, 32), torch.float32) for _ in range(3))
    k[0, 7, 0, 3] = float("nan")
    v[0, 20, 1, 3] = float("inf")
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = temporal.window_attention(q, k, v, (0, 0))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert dq[0, 7, 0].isnan().all() and dk[0, 7, 0].isnan().all() and dq[0, 20, 1].isnan().all()
    dq[0, 7, 0] = dk[0, 7, 0] = dq[0, 20, 1] = dk[0, 20, 1] = 0
    assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_rows_that_one_key_dominates(dtype):
    """Two keys of weights w, 1 - w: ds = +-w (1 - w) (dp1 - dp2), of which nothing but a relative part may be lost.  With half a
    step u: u for the rounding of ds; p times the error of delta = g . o, where the weights' roundings move o by at most
    2 u w (1 - w) (v1 - v2) and so delta by at most 2 u |ds|; u^2 |g| |o| of what two roundings leave of o.  The float32 parts
    (scores of up to 100, sums of 64) are within 2^-15 of ds.  Below the type's smallest normal value (2^-14 in float16) a step
    does not shrink any more: a rounding is off by up to half a step h there, so ds and the results by h more, a weight by h of
    the row's largest and so delta by 2 h |dp1 - dp2|, and each value that rounding left of o by h."""
    n, dim = 700, 64
    g = gen(53)
    q, k = (normal(g, (1, n, 2, dim), dtype, True, spread=2.0) for _ in range(2))
    v = normal(g, (1, n, 2, dim), dtype, True)
    up = normal(g, (1, n, 2, dim), dtype)
    got = torch.autograd.grad(temporal.window_attention(q, k, v, (1, 0)), (q, k), up)
    u, scale = torch.finfo(dtype).eps / 2, dim ** -0.5
    h = torch.finfo(dtype).tiny * u
    q, k, v, up = (f64(t)[0].transpose(0, 1) for t in (q, k, v, up))
    i = torch.arange(n)
    seen = (i[None] <= i[:, None]) & (i[None] >= i[:, None] - 1)
    p = torch.softmax((q @ k.transpose(1, 2) * scale).masked_fill(~seen, -1e300), -1)
    out, dp = p @ v, up @ v.transpose(1, 2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    off = (3 * u + 2 ** -15) * ds.abs() + p * (u * u * (up.abs() * out.abs()).sum(-1, keepdim=True))
    apart = (dp - torch.roll(dp, 1, 2)).abs().masked_fill(~seen, 0).amax(-1, keepdim=True)
    off = off + h + p * (2 * h * apart + h * up.abs().sum(-1, keepdim=True))
    off = off * (1 + 4 * u) + p * 2 ** -20 * (up.abs() @ v.abs().transpose(1, 2)).masked_fill(~seen, 0).amax(-1, keepdim=True)
    for name, a, s, o, other in (("dq", got[0], ds, off, k), ("dk", got[1], ds.transpose(1, 2), off.transpose(1, 2), q)):
        want = s @ other * scale
        bound = o @ other.abs() * scale
        within(a, want.transpose(0, 1)[None], (bound + u * (want.abs() + bound) + h).transpose(0, 1)[None], name)


# ---- plans that the sizes above do not reach ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [
    (4, 1700, 4, 2, 64, (16, 16), 1, (1700, 1, 1699, 33), False),   # float32: four waves walk a short window together
    (1, 4500, 1, 1, 32, (20, 0), 33, None, False),                  # the far queries of the sinks in 32 chunks
    (4, 1300, 6, 6, 32, (30, 0), 65, (1300, 700, 159, 0), True),    # chunks of 256
    (1, 130, 1, 1, 128, (0, 129), 0, None, False),                  # looks ahead alone
], ids=str)
def test_window_attention_plans(dtype, case):
    test_window_attention(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,slots,sinks", [(40, 1, 64, 2500, 3), (8, 2, 128, 5000, 16), (70, 2, 32, 90, 1),
                                                           (4, 4, 96, 260, 0)])
def test_window_attention_step_shares(dtype, heads, kv_heads, dim, slots, sinks):
    """Long rings and many heads that share them.  Off by at most: u for the weights' rounding and u for the result's; twice
    what float32 leaves of a score, (dim + 4) 2^-24 sum |q||k| scale; and of the sums over the slots, slots 2^-24 each."""
    g = gen(heads + slots)
    b, share, scale = 3, heads // kv_heads, dim ** -0.5
    q = normal(g, (b, heads, dim), dtype)
    k, v = normal(g, (b, kv_heads, dim), dtype), normal(g, (b, kv_heads, dim), dtype)
    kc, vc = normal(g, (b, slots, kv_heads, dim), dtype), normal(g, (b, slots, kv_heads, dim), dtype)
    lengths = torch.tensor([7 * slots, slots // 2, -3], device=DEV)
    out = f64(temporal.window_attention_step(q, k, v, kc, vc, lengths, sinks))
    assert (out[2] == 0).all()
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for s, held in ((0, slots), (1, slots // 2 + 1)):
        keys, values = (f64(c)[s, :held].repeat_interleave(share, 1).transpose(0, 1) for c in (kc, vc))
        rows = f64(q)[s][:, None]
        p = torch.softmax(rows @ keys.transpose(1, 2) * scale, -1)
        score = (dim + 4) * 2.0 ** -24 * scale * (rows.abs() @ keys.abs().transpose(1, 2)).amax()
        bound = (p @ values.abs())[:, 0] * (2 * u + 2 * score + 2 * slots * 2.0 ** -24)
        within(out[s], (p @ values)[:, 0], bound, "stream %d" % s)


def test_offsets_beyond_31_bits():
    """The last rows of tensors of more than 2^31 values give what they give by themselves."""
    g = gen(61)
    n, tail = (1 << 22) + 1024, 1024  # tokens of 8 heads of 64
    far = {name: torch.zeros(1, n, 8, 64, dtype=torch.bfloat16, device=DEV) for name in "qkvg"}
    near = {name: normal(g, (1, tail, 8, 64), torch.bfloat16) for name in "qkvg"}
    for name in "qkvg":
        far[name][:, -tail:] = near[name]
    out = {}
    for side, t in (("far", far), ("near", near)):
        leaves = [t[name].requires_grad_() for name in "qkv"]
        y = temporal.window_attention(*leaves, (63, 0))
        out[side] = [y.detach(), *torch.autograd.grad(y, leaves, t["g"])]
    for a, c in zip(out["far"], out["near"]):
        assert torch.equal(a[:, -tail + 128:], c[:, 128:])  # the first of the short sequence see fewer keys
    del out
    at = torch.arange(n, device=DEV)[:, None]
    turned = temporal.rotate_positions(far["q"].detach(), far["k"].detach(), at, (32,))
    alone = temporal.rotate_positions(near["q"].detach(), near["k"].detach(), at[-tail:], (32,))
    assert all(torch.equal(a[:, -tail:], c) for a, c in zip(turned, alone))
    del turned
    x = far["q"].detach().view(-1, 512)
    assert torch.equal(temporal.layer_norm(x)[-tail:], temporal.layer_norm(near["q"].detach().view(-1, 512)))
    # a ring of 2 x 2.1 million slots, of which the last hold something
    kc, vc = far["k"].detach().view(2, n // 2, 8, 64), far["v"].detach().view(2, n // 2, 8, 64)
    slots = n // 2
    q, k, v = (normal(g, (2, 8, 64), torch.bfloat16) for _ in range(3))
    lengths = torch.tensor([-1, slots - 1], device=DEV)
    step = temporal.window_attention_step(q, k, v, kc, vc, lengths, 4)
    assert torch.equal(kc[1, -1], k[1]) and torch.equal(vc[1, -1], v[1]) and lengths.tolist() == [-1, slots]
    keys, values = f64(kc[1, -tail:]).transpose(0, 1), f64(vc[1, -tail:]).transpose(0, 1)
    weight = torch.exp(f64(q)[1][:, None] @ keys.transpose(1, 2) / 8)
    total = weight.sum(-1) + (slots - tail)  # the other keys are zero: weights of 1, values of zero
    want = (weight @ values)[:, 0] / total
    # 2 u, and sums of 2^21 weights in float32: 32 at a time in a wave, at most 2^14 additions one after the other, 2^-24 each
    within(step[1], want, (weight @ values.abs())[:, 0] / total * (2 ** -7 + 2 ** -9), "step")
    temporal.window_cache_fill(near["k"].detach().expand(2, -1, -1, -1), near["v"].detach().expand(2, -1, -1, -1), kc, vc,
                               torch.tensor([0, tail], device=DEV), slots - 10)
    assert torch.equal(kc[1, :tail], near["k"][0]) and torch.equal(vc[1, :tail], near["v"][0])


def test_two_graphs_and_eager_calls_in_turn():
    """Workspaces belong to the graph that was captured with them."""
    g = gen(62)

    def work(seed, n, window, slots):
        g = gen(seed)
        q, k, v = (normal(g, (2, n, heads, 64), torch.bfloat16, True) for heads in (8, 2, 2))
        up = normal(g, (2, n, 8, 64), torch.bfloat16)
        kc, vc = normal(g, (2, slots, 2, 64), torch.bfloat16), normal(g, (2, slots, 2, 64), torch.bfloat16)
        held = torch.full((2,), 3 * slots, device=DEV)

        def run():
            lengths = held.clone()
            y = temporal.window_attention(q, k, v, window, 3)
            grads = torch.autograd.grad(y, (q, k, v), up)
            token = temporal.window_attention_step(q[:, 0].detach(), k[:, 0].detach(), v[:, 0].detach(), kc, vc, lengths, 3)
            return [y.detach(), *grads, token]

        return run

    jobs = [work(1, 700, (50, 0), 900), work(2, 900, (70, 20), 700)]
    want = [[t.clone() for t in job()] for job in jobs]
    side = torch.cuda.Stream()
    graphs, got = [], []
    for job in jobs:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            job()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got.append(job())
        graphs.append(graph)
    for turn in range(6):
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        eager = jobs[turn % 2]()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(eager, want[turn % 2]))
        for one, c in zip(got, want):
            assert all(torch.equal(a, e) for a, e in zip(one, c)), turn
            for t in one:
                t.zero_()
    # and two streams at once
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(side):
            a = jobs[0]()
        with torch.cuda.stream(other):
            c = jobs[1]()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, want[0])) and all(torch.equal(x, y) for x, y in zip(c, want[1]))


@pytest.mark.parametrize("width", [1000, 9000])
def test_layer_norm_of_16_bit_rows_with_float32_parameters(width):
    g = gen(63)
    x = normal(g, (37, width), torch.bfloat16, True)
    w, b = normal(g, (width,), torch.float32, True, 0.3, 1.0), normal(g, (width,), torch.float32, True, 0.3)
    up = normal(g, (37, width), torch.bfloat16)
    got = torch.autograd.grad(temporal.layer_norm(x, w, b), (x, w, b), up)
    assert [t.dtype for t in got] == [torch.bfloat16, torch.float32, torch.float32]
    _, _, grads, bounds = orc.layer_norm(f64(x), f64(w), f64(b), 1e-5, torch.bfloat16, f64(up))
    for name, a, c, e in zip(("dx", "dweight", "dbias"), got, grads, bounds):
        within(a, c, e, name)


def test_gradients_of_sinks_of_very_many_sequences():
    b, n, heads, dim, dtype = 4200, 700, 16, 8, torch.float16
    torch.manual_seed(64)
    q, k, v, up = (torch.randn(b, n, heads, dim, device=DEV, dtype=dtype) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(temporal.window_attention(*leaves, (0, 0), 2), leaves, up)
    for s in (0, b - 1):
        one = slice(s, s + 1)
        _, _, grads, bounds = orc.attention(f64(q[one]), f64(k[one]), f64(v[one]), (0, 0), 2, dtype, grad=f64(up[one]))
        for name, a, c, e in zip(("dq", "dk", "dv"), got, grads, bounds):
            within(a[one], c, e, "%s of sequence %d" % (name, s))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [
    (1, 300, 2, 1, 128, (None, 0), 3, None, False),
    (1, 600, 4, 4, 96, (100, 20), 40, (555,), True),
    (16, 500, 4, 1, 32, (50, 0), 2, None, True),     # pairs of waves for the keys, four waves for the queries
    (4, 1800, 8, 8, 16, (255, 0), 1, None, False),   # four waves for both
], ids=str)
def test_window_attention_gradients_by_pairs_of_waves(dtype, case):
    test_window_attention(dtype, case)


@pytest.mark.parametrize("case", [
    (1, 33, 1, 1, 64, (0, 0), 0, None, False),       # one tile: the second wave has none
    (2, 200, 4, 2, 40, (60, 60), 40, (200, 7), True),
    (1, 640, 8, 1, 32, (100, 20), 100, None, True),  # more tiles of sinks than of the window
    (3, 5000, 1, 1, 32, (31, 0), 1, None, False),    # 471 waves
    (3, 5700, 1, 1, 32, (31, 0), 1, None, False),    # 537: single waves again
], ids=str)
def test_window_attention_of_queries_shared_by_two_waves(case):
    test_window_attention(torch.float32, case)


def test_queries_shared_by_two_waves_pass_on_what_is_not_finite():
    q, k, v = (normal(gen(65), (1, 120, 1, 32), torch.float32) for _ in range(3))
    want, bound = orc.attention(f64(q), f64(k), f64(v), (40, 40), 0, torch.float32)
    v[0, 3, 0, 5] = float("inf")  # in the first wave's tiles and, 32 keys on, the second's
    v[0, 40, 0, 6] = float("nan")
    out = temporal.window_attention(q, k, v, (40, 40))
    assert (out[0, :44, 0, 5] == float("inf")).all() and out[0, :81, 0, 6].isnan().all()
    out = f64(out)
    out[0, :44, 0, 5], out[0, :81, 0, 6] = want[0, :44, 0, 5], want[0, :81, 0, 6]
    within(out, want, bound, "the other columns and queries")


def minus_infinity_case(dtype):
    """Sinks and keys 40 to 59 hold -inf where every query is positive, query 80 holds -inf where every key is: the scores of
    queries 45 to 59 and 80 are minus infinity alone, those of the others for these keys only."""
    n, window, sinks = 400, (5, 0), 2
    g = gen(71)
    q, k, v, up = (normal(g, (1, n, heads, 32), dtype) for heads in (2, 1, 1, 2))
    q[..., 3], k[..., 5] = q[..., 3].abs() + 0.5, k[..., 5].abs() + 0.5
    visible = torch.ones(1, n, dtype=torch.bool)
    visible[0, :2] = visible[0, 40:60] = False
    empty = torch.zeros(n, dtype=torch.bool)
    empty[45:60] = empty[80] = empty[:2] = True
    plain = [f64(t) for t in (q, k, v, up)]
    plain[0][:, 80], plain[3][:, 80] = 0, 0
    want, bound, grads, bounds = orc.attention(*plain[:3], window, sinks, dtype, visible=visible, grad=plain[3])
    want[:, 80], bound[:, 80] = 0, 0
    k[0, ~visible[0].to(DEV), :, 3] = -torch.inf
    q[0, 80, :, 5] = -torch.inf
    return q, k, v, up, window, sinks, empty, want, bound, grads, bounds


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity_alone_give_zeros_and_pass_no_gradient(dtype):
    q, k, v, up, window, sinks, empty, want, bound, grads, bounds = minus_infinity_case(dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = temporal.window_attention(*leaves, window, sinks)
    assert (out[0, empty] == 0).all()
    within(out, want, bound, "out")
    assert torch.equal(out, temporal.window_attention(*(t.detach() for t in leaves), window, sinks))
    dq, dk, dv = torch.autograd.grad(out, leaves, up)
    assert (dq[0, empty] == 0).all()
    finite = [c for c in range(32) if c != 3]  # zero times the infinite component of the sinks is a NaN
    within(dq[..., finite], grads[0][..., finite], bounds[0][..., finite], "dq")
    within(dk, grads[1], bounds[1], "dk")
    within(dv, grads[2], bounds[2], "dv")


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity_next_to_a_nan(dtype):
    q, k, v, up, window, sinks, empty, want, bound, _, _ = minus_infinity_case(dtype)
    q[0, 50, 0] = float("nan")
    out = temporal.window_attention(q, k, v, window, sinks)
    assert out[0, 50, 0].isnan().all() and (out[0, 51:60] == 0).all()
    out[0, 50, 0] = 0
    within(out, want, bound, "the others")


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_score_is_no_score_of_minus_infinity(dtype):
    q, k, v = (normal(gen(72), (1, 64, 1, 16), dtype) for _ in range(3))
    k[0, 10:14, 0, 2] = float("nan")
    q[0, 30, 0, 0], k[0, 30, 0, 0], k[0, 31, 0, 0] = -torch.inf, 1.0, float("nan")
    out = temporal.window_attention(q, k, v, (1, 1))
    nan = [9, 10, 11, 12, 13, 14, 30, 31, 32]
    assert out[0, nan].isnan().all()
    rest = [i for i in range(64) if i not in nan]
    assert torch.isfinite(out[0, rest]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,slots", [(64, 40), (32, 1500), (128, 2100)])
def test_window_attention_step_scores_of_minus_infinity(dtype, dim, slots):
    g = gen(73)
    q, k, v = normal(g, (4, 4, dim), dtype).abs() + 0.1, normal(g, (4, 2, dim), dtype), normal(g, (4, 2, dim), dtype)
    kc, vc = normal(g, (4, slots, 2, dim), dtype), normal(g, (4, slots, 2, dim), dtype)
    kc[1, :, :, 3] = k[1, :, 3] = -torch.inf  # all keys
    kc[2, ::2, :, 3] = k[2, :, 3] = -torch.inf  # every other one
    kc[3, 5, :, 3] = float("nan")
    lengths = torch.full((4,), 5 * slots + 1, device=DEV)
    out = temporal.window_attention_step(q, k, v, kc, vc, lengths)
    assert (out[1] == 0).all() and out[3].isnan().all()
    for s, kept in ((0, slice(None)), (2, f64(kc)[2, :, 0, 3].isfinite())):
        keys, values = f64(kc)[s:s + 1, kept], f64(vc)[s:s + 1, kept]
        n = keys.shape[1]
        rows = torch.zeros(1, n, 4, dim, dtype=torch.float64)
        rows[0, -1] = f64(q)[s]
        want, bound = orc.attention(rows, keys, values, (None, None), 0, dtype)
        within(out[s], want[0, -1], bound[0, -1], "stream %d" % s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_beside_one_that_is_not_finite_keep_their_bits(dtype):
    n, window, sinks = 300, (20, 6), 2
    g = gen(74)
    q, k, v, up = (normal(g, (1, n, heads, 64), dtype) for heads in (2, 1, 1, 2))

    def both(q, up):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = temporal.window_attention(*leaves, window, sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]

    clean = both(q, up)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[7, 133, 290]] = True
    q2, up2 = q.clone(), up.clone()
    q2[0, 7, 0, 1], q2[0, 133] = float("nan"), float("nan")
    up2[0, 290, 1, 0] = float("inf")
    out, dq, dk, dv = both(q2, up2)
    assert out[0, [7, 133], 0].isnan().all()
    assert torch.equal(out[0, ~bad], clean[0][0, ~bad]) and torch.equal(dq[0, ~bad], clean[1][0, ~bad])
    beyond = ~orc.seen_pairs(n, *window, sinks, None, None)[bad].any(0)  # keys that none of the three sees
    assert beyond.sum() > 200
    # those of its tiles are computed again: the same to rounding
    _, _, grads, bounds = orc.attention(f64(q), f64(k), f64(v), window, sinks, dtype, grad=f64(up))
    for name, a, c, e in zip(("dk", "dv"), (dk, dv), grads[1:], bounds[1:]):
        within(a[0, beyond], c[0, beyond], e[0, beyond], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_window_attention_step_is_a_mean_of_the_values(dtype, dim):
    """Of every 32 keys 31 have the same score, so their weights are rounded alike; the values are of one size, so a mean of them
    is off by little more than its own rounding: u |o|, and relative errors u of the weights move it by 2 u sum p |v - o| at most.
    Scores are off by (dim + 4) 2^-24 sum |q||k| scale, sums over the slots by slots 2^-24."""
    g = gen(75 + dim)
    b, heads, slots, scale = 2, 16, 3008, dim ** -0.5
    q, top, low = normal(g, (b, heads, dim), dtype), normal(g, (dim,), dtype), normal(g, (dim,), dtype)
    kc = low.expand(b, slots, 1, dim).contiguous()
    kc[:, ::32] = top
    u = torch.finfo(dtype).eps / 2
    vc = (1.5 + 2 * u * torch.randint(0, 3, (b, slots, 1, dim), generator=g)).to(dtype).to(DEV)
    k, v = kc[:, 0].clone(), vc[:, 0].clone()
    lengths = torch.full((b,), 5 * slots, device=DEV)  # the new token goes to slot 0 and is what lies there
    out = f64(temporal.window_attention_step(q, k, v, kc, vc, lengths))
    for s in range(b):
        keys, values, rows = f64(kc)[s, :, 0], f64(vc)[s, :, 0], f64(q)[s]
        p = torch.softmax(rows @ keys.T * scale, -1)
        want = p @ values
        apart = (p[:, :, None] * (values[None] - want[:, None]).abs()).sum(1)
        score = (dim + 4) * 2.0 ** -24 * scale * (rows.abs() @ keys.abs().T).amax()
        bound = u * want + 2 * u * apart * (1 + u) + want * slots * 2.0 ** -24 + 2 * score * apart
        within(out[s], want, bound, "stream %d" % s)


@pytest.mark.parametrize("size", [3e4, 1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("n,dim,window,sinks,heads,kv_heads", [(4000, 64, (None, 0), 0, 1, 1), (1500, 128, (None, None), 0, 1, 1),
                                                               (2500, 32, (900, 0), 3, 2, 1), (1200, 96, (1, 1), 0, 1, 1)])
def test_float16_gradients_of_any_size(n, dim, window, sinks, heads, kv_heads, size):
    """What the type's range does to the score gradients must not be seen in the results: each is off by half a step relative to
    itself (u), or by 2^-30 of the largest in its row (dq) or column (dk); weights likewise by u or 2^-39.  With the forward's
    weights off by u, delta = g . o is off by u sum |g| sum p |v - o|, and by u^2 |g| |o| and 2^-25 |g| of what two roundings leave
    of o.  float32: scores (dim + 4) 2^-24 sum |q||k| scale, sums 2^-24 per term.  A result is rounded to u or 2^-25."""
    dtype = torch.float16
    g = gen(n + dim)
    q, k, v = (normal(g, (1, n, h, dim), dtype, True) for h in (heads, kv_heads, kv_heads))
    up = (torch.randn((1, n, heads, dim), generator=g) * size).clamp(-6e4, 6e4).to(dtype).to(DEV)
    got = [f64(t)[0] for t in torch.autograd.grad(temporal.window_attention(q, k, v, window, sinks), (q, k, v), up)]
    u, e, scale = 2.0 ** -11, 2.0 ** -24, dim ** -0.5
    seen = orc.seen_pairs(n, *window, sinks, None, None)
    want = [torch.zeros_like(t) for t in got]
    bound = [torch.zeros_like(t) for t in got]
    for h in range(heads):
        at = h * kv_heads // heads
        qh, kh, vh, gh = f64(q)[0, :, h], f64(k)[0, :, at], f64(v)[0, :, at], f64(up)[0, :, h]
        p = torch.softmax((qh @ kh.T * scale).masked_fill(~seen, -torch.inf), -1)
        o, dp = p @ vh, gh @ vh.T
        ds = p * (dp - (gh * o).sum(-1, keepdim=True))
        x = 2 * (dim + 4) * e * scale * torch.where(seen, qh.abs() @ kh.abs().T, 0.0).amax(-1, keepdim=True) + 64 * e + n * e
        spread = (p @ vh ** 2 - o ** 2).clamp(min=0).sqrt()  # at least sum p |v - o|
        delta = (gh.abs() * (u * spread * (1 + 4 * u) + (u * u + 2 * x) * o.abs() + 2.0 ** -25)).sum(-1, keepdim=True)
        off = (u + x) * ds.abs() + p * (1 + u) * (delta + (dim + 4) * e * torch.where(seen, gh.abs() @ vh.abs().T, 0.0))
        rows, cols = (2.0 ** -30 * seen * (ds.abs() + off).amax(d, keepdim=True) for d in (1, 0))
        want[0][:, h] = scale * ds @ kh
        bound[0][:, h] = scale * (off + rows + n * e * ds.abs()) @ kh.abs()
        want[1][:, at] += scale * ds.T @ qh
        bound[1][:, at] += scale * (off + cols + n * heads * e * ds.abs()).T @ qh.abs()
        want[2][:, at] += p.T @ gh
        bound[2][:, at] += ((u + x + n * heads * e) * p + 2.0 ** -39 * seen).T @ gh.abs()
    for name, a, c, b in zip(("dq", "dk", "dv"), got, want, bound):
        over = (c.abs() + b) * (1 + u) > 65504  # beyond the type
        within(torch.where(over, 0.0, a), torch.where(over, 0.0, c), b + u * (c.abs() + b) + 2.0 ** -25, name)
        assert over.double().mean() < 0.5


def test_forward_mode_tangents_are_refused():
    """No operator has a forward-mode rule: a result without a tangent would be a derivative of zero."""
    x, w, t = torch.randn(1, 6, 2, 16, device=DEV), torch.randn(16, device=DEV), torch.randn(1, 6, 2, 16, device=DEV)
    positions, lengths = torch.zeros(6, 1, device=DEV), torch.ones(1, dtype=torch.int64, device=DEV)
    kc, vc = torch.zeros(1, 9, 2, 16, device=DEV), torch.zeros(1, 9, 2, 16, device=DEV)
    plain = temporal.window_attention(x, x, x, (2, 0))
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            d, dw = fwd.make_dual(x, t), fwd.make_dual(w, w)
            for call in (lambda: temporal.layer_norm(d), lambda: temporal.layer_norm(x, dw), lambda: temporal.layer_norm(x, w, dw),
                         lambda: temporal.rotate_positions(d, None, positions, (8,)), lambda: temporal.rotate_positions(x, d, positions, (8,)),
                         lambda: temporal.rotate_positions(x, x, fwd.make_dual(positions, positions), (8,)),
                         lambda: temporal.window_attention(d, x, x, (2, 0)), lambda: temporal.window_attention(x, d, x, (2, 0)),
                         lambda: temporal.window_attention(x, x, d, (2, 0)),
                         lambda: temporal.window_cache_fill(d, x, kc, vc, lengths), lambda: temporal.window_cache_fill(x, d, kc, vc, lengths),
                         lambda: temporal.window_attention_step(d[:, 0], x[:, 0], x[:, 0], kc, vc, lengths),
                         lambda: temporal.window_attention_step(x[:, 0], x[:, 0], d[:, 0], kc, vc, lengths)):
                with pytest.raises(_cabi.MvxError, match="tangent"):
                    call()
            assert torch.equal(temporal.window_attention(x, x, x, (2, 0)), plain)  # no tangent: as ever
    assert (kc == 0).all() and lengths.item() == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [
    (12, 1500, 4, 4, 16, (0, 0), 1490, (1500, 900) * 6, False),   # blocks of sinks alone fill the GPU
    (2, 1100, 8, 4, 32, (40, 3), 1100, (1100, 1024), True),       # every token a sink
    (1, 2300, 1, 1, 64, (7, 0), 1000, None, False),               # few chunks of many sinks
], ids=str)
def test_window_attention_gradients_of_many_sinks(dtype, case):
    q, k, v, up, lengths, visible = attention_case(case, dtype, leaf=True)
    out = temporal.window_attention(q, k, v, case[5], case[6], lengths=on_gpu(lengths), visible=on_gpu(visible))
    got = torch.autograd.grad(out, (q, k, v), up)
    for s in {0, case[0] - 1}:
        one = slice(s, s + 1)
        _, _, grads, bounds = orc.attention(f64(q)[one], f64(k)[one], f64(v)[one], case[5], case[6], dtype,
                                            None if lengths is None else lengths[one], None if visible is None else visible[one],
                                            grad=f64(up)[one])
        for name, a, c, e in zip(("dq", "dk", "dv"), got, grads, bounds):
            within(a[one], c, e, "%s of sequence %d" % (name, s))


def test_a_short_window_takes_the_batch_that_a_long_one_takes():
    b, n, heads, dim, dtype = (1 << 18) + 40, 33, 16, 8, torch.float16
    torch.manual_seed(76)
    q, k, v = (torch.randn(b, n, h, dim, device=DEV, dtype=dtype) for h in (heads, 1, 1))
    for window in ((200, 0), (2, 1)):
        out = temporal.window_attention(q, k, v, window)
        for s in (0, b // 2, b - 1):
            one = slice(s, s + 1)
            within(out[one], *orc.attention(f64(q[one]), f64(k[one]), f64(v[one]), window, 0, dtype), "sequence %d" % s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(9001, 257), (5003, 1024), (4500, 100), (9001, 64), (3000, 2000), (1100, 3000), (700, 8193), (600, 16380),
                                        (1000, 3), (300, 16385)])
def test_layer_norm_of_more_rows_than_run_at_once(dtype, rows, width):
    test_layer_norm(dtype, rows, width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [
    (1, 1201, 4, 2, 64, (8, 12, 12), True, False, torch.int32, True),
    (3, 1999, 1, 1, 40, (5, 6), True, True, torch.int64, False),
    (2, 3001, 2, 0, 36, (5, 4), True, False, torch.float32, True),
    (5, 701, 3, 1, 24, (12,), False, False, torch.int32, True),
], ids=str)
def test_rotate_positions_several_tokens_per_workgroup(dtype, case):
    if case[3]:
        test_rotate_positions(dtype, case)
        return
    b, n, h, _, d, sections, pairs, shared, ptype, _ = case
    g = gen(n)
    q, pos = normal(g, (b, n, h, d), dtype), torch.rand((b, n, len(sections)), generator=g) * 500
    out, none = temporal.rotate_positions(q, None, pos.to(DEV), sections, pairs=pairs, shared_spectrum=shared)
    assert none is None
    within(out, *orc.rotate(f64(q), pos, sections, 10000.0, shared, pairs, dtype), "q alone")
