"""Rows8, quantize8, linear8, gated8, rms_norm8 and the layers of nn that are made
of gated layers and RMS norms check their arguments before any device call.  CPU
only: tensors are metadata without buffers."""

import numpy as np
import pytest

import ember_amd as em
from ember_amd import _core, nn
from ember_amd.rows8 import Rows8
from ember_amd.tensor import Tensor

NEW = ("_rows8_write", "_rows8_read", "_rmsnorm_fwd", "_rmsnorm_fwd8", "_rmsnorm_bwd", "_linear8", "_gated_fwd", "_gated_bwd", "_gated8")


def fake(*shape):
    return Tensor._from_core(None, shape)


def fake8(rows, cols):
    return Rows8(None, None, (rows, cols))


@pytest.fixture
def calls(monkeypatch):
    """No device call is made: each notes its name and arguments."""
    made = []

    def note(name, result):
        monkeypatch.setattr(_core, name, lambda *args: made.append((name, args)) or result)
    for name in NEW:
        note(name, {"_rows8_write": (1, 2), "_rmsnorm_fwd": (1, None, 2), "_rmsnorm_fwd8": ((1, 2), None), "_rmsnorm_bwd": (1, 2),
                    "_gated_fwd": (1, 2), "_gated8": (1, 2)}.get(name, 1))
    for name in ("_uniform", "_constant", "_linear", "_gemm", "_col_sum"):
        note(name, (1, None) if name == "_linear" else 1)
    return made


def test_names():
    for name in NEW:
        assert callable(getattr(_core, name)) and name in _core.__all__
    assert {"Rows8", "quantize8", "linear8", "gated8", "rms_norm8"} <= set(em.__all__)
    assert em.linear8 is em.rows8.linear8


def test_quantize8(calls):
    with pytest.raises(TypeError):
        em.quantize8(np.zeros((2, 3)))
    for shape in ((3,), (1, 2, 3)):
        with pytest.raises(ValueError):
            em.quantize8(fake(*shape))
    assert em.quantize8(fake(3, 5)).shape == (3, 5) and em.quantize8(fake(3, 5), trans=True).shape == (5, 3)
    assert calls == [("_rows8_write", (None, 3, 5, False)), ("_rows8_write", (None, 5, 3, True))]
    assert em.quantize8(fake(3, 5)).to_tensor().shape == (3, 5)


def test_linear8(calls):
    x, w = fake8(4, 70), fake8(6, 70)
    assert em.linear8(x, w, fake(6), fake(4, 6)).shape == (4, 6)
    for a, b in ((fake(4, 70), w), (x, fake(6, 70)), (x, None)):
        with pytest.raises(TypeError):
            em.linear8(a, b)
    with pytest.raises(ValueError):
        em.linear8(x, fake8(70, 6))
    for more in (dict(b=fake(4)), dict(b=fake(1, 6)), dict(residual=fake(6, 4)), dict(residual=fake(24))):
        with pytest.raises(ValueError):
            em.linear8(x, w, **more)
    with pytest.raises(TypeError):
        em.linear8(x, w, np.zeros(6))
    assert [c[0] for c in calls] == ["_linear8"]


def test_gated8(calls):
    x, w = fake8(4, 70), fake8(6, 70)
    assert em.gated8(x, w, fake(6), "gelu").shape == (4, 3)
    with pytest.raises(TypeError):
        em.gated8(fake(4, 70), w)
    for a, b, more in ((x, fake8(5, 70), {}), (x, fake8(0, 70), {}), (x, fake8(6, 71), {}), (x, w, dict(b=fake(3))), (x, w, dict(activation="relu"))):
        with pytest.raises(ValueError):
            em.gated8(a, b, **more)
    assert [c[0] for c in calls] == ["_gated8"]


def test_rms_norm8(calls):
    x = fake(4, 8)
    y, s = em.rms_norm8(x, fake(8))
    assert y.shape == (4, 8) and s is x
    for a, gamma, more in ((fake(8), fake(8), {}), (x, fake(4), {}), (x, fake(1, 8), {}), (x, fake(8), dict(residual=fake(8, 4)))):
        with pytest.raises(ValueError):
            em.rms_norm8(a, gamma, **more)
    with pytest.raises(TypeError):
        em.rms_norm8(x, np.zeros(8))
    assert [c[0] for c in calls] == ["_rmsnorm_fwd8"]


def test_gated_functions(calls):
    for x, w, more in ((fake(4, 8), fake(8, 7), {}), (fake(4, 8), fake(7, 8), {}), (fake(4, 8), fake(8, 0), {}),
                       (fake(4, 8), fake(8, 6), dict(b=fake(3))), (fake(4, 8), fake(8, 6), dict(activation="tanh")), (fake(8), fake(8, 6), {})):
        with pytest.raises(ValueError):
            nn.gated(x, w, **more)
    for dy, w, pre in ((fake(4, 8), fake(3, 7), fake(4, 6)), (fake(4, 8), fake(3, 8), fake(4, 3)), (fake(4, 8), fake(3, 8), fake(5, 6))):
        with pytest.raises(ValueError):
            nn.gated_grad(dy, w, pre)
    h, pre = nn.gated(fake(4, 8), fake(8, 6))
    assert h.shape == (4, 3) and pre.shape == (4, 6) and nn.gated_grad(fake(4, 8), fake(3, 8), pre).shape == (4, 6)


def test_layers(calls):
    with pytest.raises(ValueError):
        nn.GatedFeedForward(8, 6, activation="relu")
    for d, hidden in ((0, 6), (8, 0)):
        with pytest.raises(ValueError):
            nn.GatedFeedForward(d, hidden)
    layer = nn.GatedFeedForward(8, 6)
    assert [p.shape for p in layer.parameters()] == [(8, 12), (12,), (6, 8), (8,)] and layer.gradients() == [None] * 4
    assert [p.shape for p in nn.GatedFeedForward(8, 6, bias=False).parameters()] == [(8, 12), (6, 8)]
    with pytest.raises(RuntimeError):
        layer.backward(fake(2, 8))
    layer(fake(2, 8))
    assert layer.backward(fake(2, 8)).shape == (2, 8) and [g.shape for g in layer.gradients()] == [(8, 12), (12,), (6, 8), (8,)]
    layer(fake(2, 8), training=False)
    with pytest.raises(RuntimeError):
        layer.backward(fake(2, 8))
    norm = nn.RMSNorm(8)
    with pytest.raises(RuntimeError):
        norm.backward(fake(2, 8))
    with pytest.raises(ValueError):
        norm.forward(fake(2, 8), residual=fake(1, 8))
    norm(fake(2, 8))
    assert norm.backward(fake(2, 8)).shape == (2, 8) and norm.gradients()[0].shape == (8,)


def test_blocks(calls):
    for more in (dict(norm="batch"), dict(gated="relu"), dict(hidden=0)):
        with pytest.raises(ValueError):
            nn.DecoderBlock(64, 2, **more)
    shapes = lambda **kw: [p.shape for p in nn.DecoderBlock(64, 2, **kw).parameters()]  # noqa: E731
    assert shapes() == [(64,), (64,), (64, 192), (192,), (64, 64), (64,), (64,), (64,), (64, 256), (256,), (256, 64), (64,)]
    assert shapes(hidden=100)[8:] == [(64, 100), (100,), (100, 64), (64,)] and shapes(mlp_ratio=2)[8:] == [(64, 128), (128,), (128, 64), (64,)]
    assert shapes(norm="rms", gated="silu", hidden=100) == [(64,), (64, 192), (192,), (64, 64), (64,), (64,), (64, 200), (200,), (100, 64), (64,)]
    with pytest.raises(ValueError):
        nn.DecoderBlock(64, 2, causal=False).quantize8()
    block = nn.DecoderBlock(64, 2, norm="rms", gated="gelu").quantize8()
    assert (block.w_qkv.shape, block.w_o.shape, block.w_1.shape, block.w_2.shape) == ((192, 64), (64, 64), (512, 64), (64, 256))


@pytest.mark.parametrize("kind", [dict(norm="rms", gated="gelu"), {}])
def test_an_8_bit_block_needs_its_block_no_longer(calls, kind):
    import gc
    import weakref

    block = nn.DecoderBlock(64, 2, **kind)
    shapes = [p.shape for p in block.parameters()]
    block8 = block.quantize8()
    assert [p.shape for p in block.parameters()] == shapes
    held = {id(t) for o in (block8, block8.ln1, block8.ln2) for t in vars(o).values() if isinstance(t, Tensor)}
    assert held and not held & {id(t) for t in block.parameters()}
    gone = weakref.ref(block)
    del block
    gc.collect()
    assert gone() is None


def test_binding_checks_its_arguments():
    for name, args in (("_rows8_write", (None, 1, 1, False)), ("_rows8_read", (None,)), ("_rows8_read", ((None, None, 1, 1),)),
                       ("_rmsnorm_fwd", (None, None, None, 1, 4, 0.0)), ("_rmsnorm_fwd8", (None, None, None, 1, 4, 0.0)),
                       ("_rmsnorm_bwd", (None, None, None, None, None, 1, 4)), ("_linear8", ((1, 2), (1, 2), None, None, 0)),
                       ("_gated_fwd", (None, None, None, 1, 1, 1, 1, True)), ("_gated_bwd", (None, None, None, 1, 1, 1, 1)), ("_gated8", (1, 2, None, 1))):
        with pytest.raises(TypeError):
            getattr(_core, name)(*args)
