"""CPU checks of the sequence operators: refusals that need no GPU, the argument checks of their C entry points, and the oracle
itself (its gradients against differences and against autograd of the plain formula)."""
import ctypes

import pytest
import torch

import temporal_oracle as orc
from poseestimation_amd import _cabi, temporal

BAD, UNSUPPORTED, OK = _cabi.MVX_ERR_INVALID_ARGUMENT, _cabi.MVX_ERR_UNSUPPORTED, _cabi.MVX_OK
S3 = ctypes.c_int64 * 3
I32 = ctypes.c_int32
SOME = 0x1000  # an address that the checks see and nothing reads


def test_cpu_tensors_and_other_types_are_refused():
    t = torch.zeros(1, 4, 2, 16)
    for call in (lambda: temporal.layer_norm(t), lambda: temporal.rotate_positions(t, None, torch.zeros(4, 1), (8,)),
                 lambda: temporal.window_attention(t, t, t, (1, 1)),
                 lambda: temporal.window_cache_fill(t, t, t, t, torch.zeros(1, dtype=torch.int64)),
                 lambda: temporal.window_attention_step(t[:, 0], t[:, 0], t[:, 0], t, t, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(_cabi.MvxError, match="HIP device only"):
            call()
    with pytest.raises(TypeError):
        temporal.layer_norm([1.0])
    with pytest.raises(TypeError):
        temporal.window_attention(None, t, t, (1, 1))


def test_layer_norm_argument_checks():
    lib = _cabi.load()
    f = lib.mvx_layer_norm
    assert f(None, None, None, 0, 0, 0, 64, 1e-5, None, None, None) == OK
    assert f(None, None, None, 0, 0, 3, 64, 1e-5, None, None, None) == BAD
    assert f(SOME, None, None, 7, 0, 3, 64, 1e-5, SOME, None, None) == BAD
    assert f(SOME, None, None, 0, 0, 3, 0, 1e-5, SOME, None, None) == BAD
    assert f(SOME, None, None, 0, 0, -1, 64, 1e-5, SOME, None, None) == BAD
    assert f(SOME, None, None, 0, 0, 1 << 31, 64, 1e-5, SOME, None, None) == UNSUPPORTED
    g = lib.mvx_layer_norm_backward
    assert lib.mvx_layer_norm_backward_workspace_bytes(0, 0, 64) == 0
    need = lib.mvx_layer_norm_backward_workspace_bytes(1, 65536, 1024)
    assert need > 0 and need % (2 * 1024 * 4) == 0  # whole rows of partial sums
    assert g(SOME, SOME, None, SOME, 1, 0, 65536, 1024, None, None, None, None, 0, None) == OK  # nothing asked for
    assert g(SOME, SOME, None, None, 1, 0, 65536, 1024, SOME, None, None, None, 0, None) == BAD
    assert g(SOME, SOME, None, SOME, 1, 0, 65536, 1024, SOME, SOME, None, SOME, need - 1, None) == _cabi.MVX_ERR_WORKSPACE
    assert b"workspace" in lib.mvx_last_error()


def test_rotary_argument_checks():
    lib = _cabi.load()

    def call(q=SOME, heads=2, k_heads=0, dtype=0, seqs=1, tokens=4, dim=16, pos_type=0, axes=2, sections=(4, 4), base=1e4):
        return lib.mvx_rotate_positions(q, S3(0, 32, 16), heads, None, None, k_heads, dtype, seqs, tokens, dim, SOME, pos_type, 0,
                                        axes, (I32 * len(sections))(*sections), base, 0, 0, 0, SOME, None, None)

    assert call(tokens=0) == OK and call(seqs=0) == OK
    assert call(q=None) == BAD and call(heads=0) == BAD and call(dim=0) == BAD and call(tokens=-1) == BAD
    assert call(k_heads=1) == BAD  # no k given
    assert call(pos_type=4) == BAD and call(axes=0) == BAD and call(axes=5, sections=(1,) * 5) == BAD
    assert call(sections=(4, 5)) == BAD and call(sections=(0, 0)) == BAD and call(sections=(-1, 4)) == BAD
    assert call(base=0.0) == BAD and call(base=float("inf")) == BAD and call(base=float("nan")) == BAD
    assert call(dim=1000, sections=(100, 100)) == UNSUPPORTED
    assert call(seqs=1 << 20, tokens=1 << 20) == UNSUPPORTED
    assert call(dtype=3) == BAD


def test_attention_argument_checks():
    lib = _cabi.load()
    st = S3(4 * 2 * 16, 2 * 16, 16)

    def call(q=SOME, strides=st, dtype=0, seqs=1, tokens=4, heads=2, kv=2, dim=16, left=1, right=1, sinks=0, scale=1.0, out=SOME):
        return lib.mvx_window_attention(q, strides, SOME, st, SOME, st, dtype, seqs, tokens, heads, kv, dim, left, right, sinks, scale,
                                        None, None, out, None, None)

    assert call(seqs=0) == OK and call(tokens=0) == OK
    assert call(q=None) == BAD and call(out=None) == BAD and call(q=SOME + 4) == BAD and call(strides=S3(128, 32, 17)) == BAD
    assert call(heads=3) == BAD and call(heads=0) == BAD and call(kv=0) == BAD and call(dtype=5) == BAD
    assert call(dim=12) == BAD and call(dim=0) == BAD and call(dim=136) == UNSUPPORTED
    assert call(left=-1) == BAD and call(right=-1) == BAD and call(sinks=-1) == BAD
    assert call(scale=0.0) == BAD and call(scale=float("nan")) == BAD and call(scale=float("inf")) == BAD
    assert call(tokens=(1 << 30) + 1) == UNSUPPORTED and call(tokens=1 << 30, seqs=1 << 20) == UNSUPPORTED
    need = lib.mvx_window_attention_backward_workspace_bytes(1, 1000, 2, 2, 16, 100, 4)
    assert need >= 2 * 1000 * 4
    assert lib.mvx_window_attention_backward(SOME, st, SOME, st, SOME, st, SOME, SOME, SOME, st, 0, 1, 1000, 2, 2, 16, 100, 0, 4, 1.0,
                                             None, None, SOME, SOME, SOME, SOME, need - 1, None) == _cabi.MVX_ERR_WORKSPACE
    assert lib.mvx_window_attention_backward(SOME, st, SOME, st, SOME, st, SOME, None, SOME, st, 0, 1, 1000, 2, 2, 16, 100, 0, 4, 1.0,
                                             None, None, SOME, SOME, SOME, SOME, need, None) == BAD


def test_ring_argument_checks():
    lib = _cabi.load()

    def step(q=SOME, dtype=0, seqs=1, heads=2, kv=2, dim=16, window=8, sinks=1, scale=1.0, cache=SOME, ws=1 << 20):
        return lib.mvx_window_attention_step(q, SOME, SOME, dtype, seqs, heads, kv, dim, window, sinks, scale, cache, SOME, SOME,
                                             SOME, SOME, ws, None)

    assert step(seqs=0) == OK
    assert step(q=None) == BAD and step(cache=None) == BAD and step(cache=SOME + 8) == BAD and step(dtype=3) == BAD
    assert step(window=0) == BAD and step(sinks=-1) == BAD and step(heads=3) == BAD and step(dim=20) == BAD and step(scale=-1.0) == BAD
    assert step(dim=256) == UNSUPPORTED and step(seqs=70000) == UNSUPPORTED
    assert step(ws=3, window=1 << 20) == _cabi.MVX_ERR_WORKSPACE
    st = S3(4 * 2 * 16, 2 * 16, 16)

    def fill(k=SOME, strides=st, tokens=4, window=8, sinks=1, cache=SOME):
        return lib.mvx_window_cache_fill(k, strides, SOME, st, 0, SOME, 1, tokens, 2, 16, window, sinks, cache, SOME, None)

    assert fill(tokens=0) == OK
    assert fill(k=None) == BAD and fill(strides=S3(128, 33, 16)) == BAD and fill(tokens=-1) == BAD and fill(window=0) == BAD
    assert fill(cache=None) == BAD


def test_oracle_gradients_against_differences():
    g = torch.Generator()
    g.manual_seed(1)
    q, k, v, up = (torch.randn(1, 9, h, 8, generator=g, dtype=torch.float64) for h in (2, 1, 1, 2))
    visible = torch.ones(1, 9, dtype=torch.bool)
    visible[0, 4] = False
    how = dict(window=(3, 1), sinks=1, dtype=torch.float32, lengths=torch.tensor([8]), visible=visible)
    _, _, grads, _ = orc.attention(q, k, v, grad=up, **how)
    for t, grad in zip((q, k, v), grads):
        for at in ((0, 0, 0, 0), (0, 4, 0, 3), (0, 7, 0, 7), (0, 8, 0, 1)):
            keep, value = t[at].clone(), []
            for d in (1e-5, -1e-5):
                t[at] = keep + d
                value.append((orc.attention(q, k, v, **how)[0] * up).sum())
            t[at] = keep
            assert abs((value[0] - value[1]) / 2e-5 - grad[at]) < 1e-8
    x, w, b, up = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 7), (7,), (7,), (3, 7)))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (7,), leaves[1], leaves[2], 1e-5)
    mine = orc.layer_norm(x, w, b, 1e-5, torch.float32, up)
    assert torch.allclose(mine[0], y.detach(), rtol=1e-12, atol=1e-12)
    for a, c in zip(mine[2], torch.autograd.grad(y, leaves, up)):
        assert torch.allclose(a, c, rtol=1e-10, atol=1e-12)


def test_oracle_ring_matches_the_window():
    """What the ring of a stream holds is what its next token sees."""
    window, sinks, n = 5, 3, 23
    tokens = torch.arange(1.0, n + 1, dtype=torch.float64).view(1, n, 1, 1)
    for length in range(1, n + 1):
        ring = torch.zeros(1, sinks + window, 1, 1, dtype=torch.float64)
        orc.fill(tokens, ring, torch.tensor([length]), sinks)
        seen = orc.seen_pairs(length, window - 1, 0, sinks, None, None)[-1]
        assert sorted(ring[ring > 0].tolist()) == tokens[0, :length, 0, 0][seen].tolist()


def test_a_ring_whose_size_passes_64_bits_is_refused():
    lib = _cabi.load()
    big = (1 << 63) - 1
    assert lib.mvx_window_attention_step_workspace_bytes(0, 1, 1, 1, 8, big, big) == 0
    for window, sinks in ((big, 1), (1, big), (big, big)):
        assert lib.mvx_window_attention_step(SOME, SOME, SOME, 0, 1, 1, 1, 8, window, sinks, 1.0, SOME, SOME, SOME, SOME, None, 0,
                                             None) == UNSUPPORTED


def test_sections_of_parts_of_pairs_are_refused():
    t, positions = torch.zeros(1, 4, 2, 16), torch.zeros(4, 2)
    for sections in ((4.5, 3), (3.999, 4), ("4", "4"), (4, True + 0.5)):
        with pytest.raises(ValueError, match="whole numbers"):
            temporal.rotate_positions(t, None, positions, sections)
    for sections in ((4, 4), (4.0, 4.0), [4, 4], torch.tensor([4, 4])):
        with pytest.raises(_cabi.MvxError, match="HIP device only"):  # taken; what is refused is the CPU tensor
            temporal.rotate_positions(t, None, positions, sections)


def test_backward_workspace_stays_small_with_many_sinks():
    """The sums of the sinks' far queries (256 bytes per chunk of 32 sinks and value of a head): at most those of 2048 chunks, or a
    byte per token and value, or one chunk for each of up to three blocks of sinks."""
    size = _cabi.load().mvx_window_attention_backward_workspace_bytes
    for seqs in (1, 6, 300):
        for n in (300, 8192, 100000):
            for kv_heads, dim in ((1, 128), (8, 128), (16, 64), (4, 40)):
                for left in (0, 255, n // 2):
                    for sinks in (0, 1, 33, 130, 1000, n):
                        rows, wide = seqs * kv_heads, (dim + 31) // 32 * 32
                        sums = size(seqs, n, kv_heads, kv_heads, dim, left, sinks) - 4 * ((rows * n + 3) // 4 * 4)
                        assert 0 <= sums <= wide * max(2048 * 256, rows * n, rows * 256 * min(3, (sinks + 31) // 32)), (seqs, n, kv_heads, dim, left, sinks)
