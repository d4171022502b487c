"""nn.RMSNorm, nn.GatedFeedForward and decoder blocks made of them, in training and
decoding with and without matrices in 8 bits, against float64."""

import numpy as np
import pytest

import ember_amd as em
import gpu_helpers as G
from ember_amd import _core, capi, nn, optim
from feedforward_helpers import ff
from oracle import decoder
from test_serving_gpu import cached_attention
from tolerance import assert_north_star

pytestmark = pytest.mark.gpu


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def wide(t):
    return t.to_np().astype(np.float64)


def test_quantize8_round_trip():
    x = normal(np.random.default_rng(0), 7, 300)
    for trans in (False, True):
        m = em.quantize8(em.Tensor(x), trans)
        want = np.ascontiguousarray(x.T) if trans else x
        codes, scales = ff.quantise8(want)
        np.testing.assert_array_equal(m.to_tensor().to_np(), ff.values8(codes, scales, want.shape[1]))
        assert m.nbytes == codes.size + scales.size
    assert em.quantize8(em.Tensor._from_core(_core._Tensor(0), (0, 5))).to_tensor().shape == (0, 5)


def test_functions_of_8_bit_matrices():
    """Small whole numbers, on which every step but the gate is exact."""
    rng = np.random.default_rng(1)
    x, w = rng.integers(-15, 16, (5, 200)).astype(np.float32), rng.integers(-15, 16, (200, 12)).astype(np.float32)
    b, r = rng.integers(-9, 9, 12).astype(np.float32), rng.integers(-9, 9, (5, 12)).astype(np.float32)
    x8, w8 = em.quantize8(em.Tensor(x)), em.quantize8(em.Tensor(w), trans=True)
    np.testing.assert_array_equal(em.linear8(x8, w8, em.Tensor(b), em.Tensor(r)).to_np(), x @ w + b + r)
    far = np.float32([4096] * 6 + [-1, 0, 1, 2, 3, -4])  # gates of 4096 pass what they gate unchanged
    h = em.gated8(em.quantize8(em.Tensor(np.ones((3, 200), np.float32))), em.quantize8(em.Tensor(np.zeros((12, 200), np.float32))), em.Tensor(far), "silu")
    np.testing.assert_array_equal(h.to_tensor().to_np(), np.tile(4096 * far[6:], (3, 1)))
    y, s = em.rms_norm8(em.Tensor(np.full((2, 64), 3, np.float32)), em.Tensor(np.full(64, 2, np.float32)), 0.0, em.Tensor(np.full((2, 64), -1, np.float32)))
    np.testing.assert_array_equal(s.to_np(), 2)
    np.testing.assert_array_equal(y.to_tensor().to_np(), 2)


def test_binding_refuses_other_sizes():
    t = _core._Tensor
    a, w = (t(3 * 64), t(3), 3, 200), (t(5 * 64), t(5), 5, 200)  # 256 bytes of codes and 4 of scales a row
    _core._linear8(a, w, None, None, 0)
    bad = [
        lambda: _core._rows8_read((t(3 * 64), t(2), 3, 200)), lambda: _core._rows8_read((t(3 * 50), t(3), 3, 200)),
        lambda: _core._rows8_read((t(0), t(0), -1, 200)), lambda: _core._rows8_read((t(0), t(0), 0, 0)), lambda: _core._rows8_read((t(0), t(0), 0, 2 ** 24)),
        lambda: _core._rows8_write(t(15), 4, 4, False), lambda: _core._rows8_write(t(16), 2 ** 27, 4, False),
        lambda: _core._linear8(a, (t(5 * 32), t(5), 5, 100), None, None, 0), lambda: _core._linear8(a, w, t(3), None, 0),
        lambda: _core._linear8(a, w, None, t(14), 0), lambda: _core._linear8(a, w, None, None, 2),
        lambda: _core._gated8(a, w, None, 2), lambda: _core._gated8(a, (t(4 * 64), t(4), 4, 200), t(2), 2), lambda: _core._gated8(a, (t(4 * 64), t(4), 4, 200), None, 0),
        lambda: _core._rmsnorm_fwd(t(8), t(4), t(4), 2, 4, 0.0), lambda: _core._rmsnorm_fwd(t(8), None, t(3), 2, 4, 0.0), lambda: _core._rmsnorm_fwd(t(8), None, t(4), 2, 4, -1.0),
        lambda: _core._rmsnorm_fwd(t(6), None, t(3), 2, 3, 0.0), lambda: _core._rmsnorm_fwd8(t(8), t(9), t(4), 2, 4, 0.0), lambda: _core._rmsnorm_fwd8(t(7), None, t(4), 2, 4, 0.0),
        lambda: _core._rmsnorm_bwd(t(8), t(4), t(1), t(8), None, 2, 4), lambda: _core._rmsnorm_bwd(t(8), t(4), t(2), t(8), t(4), 2, 4),
        lambda: _core._gated_fwd(t(8), t(23), None, 2, 3, 4, 1, True), lambda: _core._gated_fwd(t(8), t(24), t(3), 2, 3, 4, 1, True), lambda: _core._gated_fwd(t(8), t(24), None, 2, 3, 4, 0, True),
        lambda: _core._gated_bwd(t(8), t(12), t(6), 2, 3, 4, 1), lambda: _core._gated_bwd(t(8), t(12), t(12), 2, 3, 4, 3),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("shape", [(5, 64), (2, 9, 1028)])
def test_rms_norm_layer(shape):
    rng = np.random.default_rng(2)
    d = shape[-1]
    x, r, g, past = (normal(rng, *shape) for _ in range(4))
    layer = nn.RMSNorm(d)
    layer.gamma = em.Tensor(normal(rng, d))
    y = layer.forward(em.Tensor(x), residual=em.Tensor(r))
    np.testing.assert_array_equal(layer.sum.to_np(), x + r)
    gamma, rows = layer.gamma.to_np(), lambda a: a.reshape(-1, d)
    ref, rstd = ff.rmsnorm_fwd(rows(x + r), gamma, layer.eps)
    ref_dx, ref_dgamma = ff.rmsnorm_bwd(rows(x + r), gamma, rstd, rows(g), rows(past))
    dx = layer.backward(em.Tensor(g), em.Tensor(past))
    assert y.shape == dx.shape == shape
    assert_north_star(rows(y.to_np()), ref)
    assert_north_star(rows(dx.to_np()), ref_dx)
    assert_north_star(layer.gradients()[0].to_np(), ref_dgamma)
    assert_north_star(rows(layer(em.Tensor(x)).to_np()), ff.rmsnorm_fwd(rows(x), gamma, layer.eps)[0])
    with pytest.raises(ValueError):
        layer(em.Tensor(normal(rng, 2, d + 4)))


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("n, d, hidden", [(1, 64, 170), (50, 96, 100), (300, 128, 341)])
def test_gated_feed_forward(n, d, hidden, bias, activation):
    rng = np.random.default_rng(n + hidden)
    em.random.seed(n)
    layer = nn.GatedFeedForward(d, hidden, activation, bias)
    if bias:
        layer.b_in, layer.b_out = em.Tensor(normal(rng, 2 * hidden)), em.Tensor(normal(rng, d))
    x, g = em.Tensor(normal(rng, n, d)), em.Tensor(normal(rng, n, d))
    y = layer(x)
    dx = layer.backward(g)
    at = [wide(p) for p in layer.parameters()]
    w_in, b_in, w_out, b_out = at if bias else (at[0], 0, at[1], 0)
    x64, g64 = wide(x), wide(g)
    pre = x64 @ w_in + b_in
    h = ff.gate(activation, pre)
    dpre = ff.gate_bwd(activation, g64 @ w_out.T, pre)
    assert_north_star(y.to_np(), h @ w_out + b_out)
    grads = [x64.T @ dpre, dpre.sum(0), h.T @ g64, g64.sum(0)]
    for i, (got, want) in enumerate(zip([dx, *layer.gradients()], [dpre @ w_in.T, *(grads if bias else grads[::2])])):
        assert_north_star(got.to_np(), want, f"gradient {i}")
    np.testing.assert_array_equal(layer(x, training=False).to_np(), y.to_np())


def block64(block, x, dy, B, S):
    """The block in float64: y, and the gradients of x and of the parameters."""
    rest = [wide(p) for p in block.parameters()]
    x, dy = wide(x), wide(dy)

    def norm(t):
        gamma = rest.pop(0)
        if block.norm == "rms":
            y, rstd = ff.rmsnorm_fwd(t, gamma, 1e-5)
            return y, lambda g: ff.rmsnorm_bwd(t, gamma, rstd, g)
        y, kept = decoder._ln(t, gamma, rest.pop(0))
        return y, lambda g: decoder._ln_bwd(g, gamma, kept)
    h1, back1 = norm(x)
    w_qkv, b_qkv, w_o, b_o = rest[:4]
    del rest[:4]
    o, kept = decoder._attn(h1 @ w_qkv + b_qkv, B, S, block.h, block.causal)
    x2 = x + o @ w_o + b_o
    h2, back2 = norm(x2)
    w_1, b_1, w_2, b_2 = rest
    u = h2 @ w_1 + b_1
    a = ff.gate(block.gated, u) if block.gated else ff.activate("gelu", u)[0]
    da = dy @ w_2.T
    du = ff.gate_bwd(block.gated, da, u) if block.gated else da * ff.activate("gelu", u)[1]
    dh2, *norm2 = back2(du @ w_1.T)
    dx2 = dy + dh2
    dqkv = decoder._attn_bwd(dx2 @ w_o.T, kept, B, S, block.h)
    dh1, *norm1 = back1(dqkv @ w_qkv.T)
    return x2 + a @ w_2 + b_2, [dx2 + dh1, *norm1, h1.T @ dqkv, dqkv.sum(0), o.T @ dx2, dx2.sum(0),
                                *norm2, h2.T @ du, du.sum(0), a.T @ dy, dy.sum(0)]


@pytest.mark.parametrize("kind", [dict(norm="rms", gated="silu", hidden=171), dict(norm="rms", gated="gelu"), dict(norm="rms"), dict(gated="silu"), {}])
@pytest.mark.parametrize("causal", [True, False])
def test_decoder_block(kind, causal):
    B, S, H, d = 2, 40, 2, 64
    rng = np.random.default_rng(3)
    em.random.seed(4)
    block = nn.DecoderBlock(d, H, 4, causal, **kind)
    for p in block.parameters():  # no zeros or ones
        p._adopt(em.Tensor(p.to_np() + 0.1 * normal(rng, *p.shape)))
    x, g = em.Tensor(normal(rng, B * S, d)), em.Tensor(normal(rng, B * S, d))
    G.say(f"decoder block {kind} causal={causal}")
    y = block(x, B, S)
    dx = block.backward(g)
    ref, grads = block64(block, x, g, B, S)
    assert_north_star(y.to_np(), ref, "y")
    assert len(grads) == 1 + len(block.gradients())
    for i, (got, want) in enumerate(zip([dx, *block.gradients()], grads)):
        assert_north_star(got.to_np(), want, f"gradient {i}")


def test_training_steps():
    """A few steps of a block of both: every parameter moves, and stays finite."""
    em.random.seed(5)
    rng = np.random.default_rng(5)
    block = nn.DecoderBlock(64, 2, norm="rms", gated="silu", hidden=170)
    before = [p.to_np() for p in block.parameters()]
    opt, mse = optim.Adam(block.parameters(), lr=1e-3), em.loss.MSELoss()
    x, target = em.Tensor(normal(rng, 60, 64)), em.Tensor(normal(rng, 60, 64))
    for _ in range(3):
        mse(block(x, 2, 30), target)
        block.backward(mse.backward())
        opt.apply(block.gradients())
    for p, b in zip(block.parameters(), before):
        assert np.isfinite(p.to_np()).all() and (p.to_np() != b).any()


def decode64(block, weights, x, start, count, cached, T):
    """decode in float64 with the given matrices, its attention over what the cache holds."""
    w_qkv, w_o, w_1, w_2 = weights

    def norm(x, n):
        if block.norm == "rms":
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + n.eps) * wide(n.gamma)
        return (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + n.eps) * wide(n.gamma) + wide(n.beta)
    x = x.astype(np.float64)
    qkv = (norm(x, block.ln1) @ w_qkv + wide(block.b_qkv)).reshape(len(start), T, 3, block.h, block.d // block.h)
    o = cached_attention(qkv[:, :, 0], *cached, start, count).reshape(x.shape)
    x2 = x + o @ w_o + wide(block.b_o)
    u = norm(x2, block.ln2) @ w_1 + wide(block.b_1)
    return x2 + (ff.gate(block.gated, u) if block.gated else ff.activate("gelu", u)[0]) @ w_2 + wide(block.b_2)


KINDS = [dict(norm="rms", gated="silu", hidden=200), dict(norm="rms", gated="gelu"), dict(gated="silu"), {}]
STEPS = ((21, [21, 9]), (1, None), (1, None), (3, [3, 0]))


def some_block(kind, d=128, heads=2):
    em.random.seed(6)
    rng = np.random.default_rng(7)
    block = nn.DecoderBlock(d, heads, **kind)
    for p in block.parameters():
        p._adopt(em.Tensor(p.to_np() + 0.05 * normal(rng, *p.shape)))
    return block, rng


@pytest.mark.parametrize("kind", KINDS)
def test_decode(kind):
    block, rng = some_block(kind)
    cache = block.make_cache(2, 64, page_size=16)
    for T, count in STEPS:
        start = cache.lengths
        x = normal(rng, 2 * T, 128)
        y = block.decode(em.Tensor(x), cache, count).to_np()
        weights = [getattr(block, n).to_np().astype(np.float64) for n in ("w_qkv", "w_o", "w_1", "w_2")]
        assert_north_star(y, decode64(block, weights, x, start, count or [T, T], [t.to_np() for t in cache.read()], T))


@pytest.mark.parametrize("kind", KINDS)
def test_decode_in_8_bits(kind):
    """Bit for bit the public functions in turn, and near float64 with the weights
    that the 8-bit matrices hold: what is left is the rounding of four inputs of
    products to at most 2^-4 of each element, which passes on to the branches' sums
    with signs of its own; four times 2^-4 of the branches' size covers it."""
    block, rng = some_block(kind)
    block8 = block.quantize8()
    assert block8.nbytes < 0.27 * sum(4 * np.prod(w.shape) for w in (block.w_qkv, block.w_o, block.w_1, block.w_2))
    cache, twin = block8.make_cache(2, 64, page_size=16), block8.make_cache(2, 64, page_size=16)
    w = [em.quantize8(getattr(block, n), trans=True) for n in ("w_qkv", "w_o", "w_1", "w_2")]
    weights = [m.to_tensor().to_np().astype(np.float64).T for m in w]
    for T, count in STEPS:
        start = cache.lengths
        x = normal(rng, 2 * T, 128)
        G.say(f"DecoderBlock8.decode {kind} T={T}")
        y = block8.decode(em.Tensor(x), cache, count).to_np()
        tx = em.Tensor(x)

        def normed(t, n):
            if block.norm == "rms":
                return em.rms_norm8(t, n.gamma, n.eps)[0]
            return em.quantize8(n.forward(t))
        qkv = em.linear8(normed(tx, block.ln1), w[0], block.b_qkv).to_np().reshape(2, T, 3, 2, 64)
        q, k, v = (em.Tensor(np.ascontiguousarray(qkv[:, :, i])) for i in range(3))
        twin.write(k, v, count)
        o = twin.attention(q)[0].to_np().reshape(2 * T, 128)
        x2 = em.linear8(em.quantize8(em.Tensor(o)), w[1], block.b_o, tx)
        h2 = normed(x2, block.ln2)
        a = em.gated8(h2, w[2], block.b_1, block.gated) if block.gated else em.quantize8(em.linear8(h2, w[2], block.b_1, gelu=True))
        np.testing.assert_array_equal(y, em.linear8(a, w[3], block.b_2, x2).to_np())
        ref = decode64(block, weights, x, start, count or [T, T], [t.to_np() for t in cache.read()], T)
        assert np.linalg.norm(y - ref) <= 4 * 2.0 ** -4 * np.linalg.norm(ref - x)
    assert block8.decode(em.Tensor._from_core(_core._Tensor(0), (0, 128)), cache).shape == (0, 128)


def test_8_bit_block_keeps_its_weights():
    """A block8 is of the block's matrices when it was made, whatever becomes of them."""
    block, rng = some_block(KINDS[0])
    block8 = block.quantize8()
    x = em.Tensor(normal(rng, 3, 128))
    y = block8.decode(x, block8.make_cache(3, 4)).to_np()
    for w in (block.w_qkv, block.w_o, block.w_1, block.w_2):
        w._adopt(em.Tensor(np.zeros(w.shape, np.float32)))
    np.testing.assert_array_equal(block8.decode(x, block8.make_cache(3, 4)).to_np(), y)


@pytest.mark.parametrize("kind", KINDS)
def test_8_bit_block_keeps_all_of_its_weights(kind):
    """Biases and norms too: trained on in place, set anew and reset, the block changes
    and its block8 does not."""
    block, rng = some_block(kind)
    block8 = block.quantize8()
    x = em.Tensor(normal(rng, 3, 128))
    y = block8.decode(x, block8.make_cache(3, 4)).to_np()
    before = block.decode(x, block.make_cache(3, 4)).to_np()
    grads = [em.Tensor(np.full(p.shape, 0.5, np.float32)) for p in block.parameters()]
    optim.SGD(block.parameters(), lr=1.0).apply(grads)
    assert (block.decode(x, block.make_cache(3, 4)).to_np() != before).any()
    np.testing.assert_array_equal(block8.decode(x, block8.make_cache(3, 4)).to_np(), y)
    for p in block.parameters():
        p._adopt(em.Tensor(np.full(p.shape, 3, np.float32)))
    np.testing.assert_array_equal(block8.decode(x, block8.make_cache(3, 4)).to_np(), y)
    block.reset()
    block.norm, block.gated = "layer", None
    np.testing.assert_array_equal(block8.decode(x, block8.make_cache(3, 4)).to_np(), y)


def test_decode_leaves_training_alone():
    block, rng = some_block(KINDS[0], 64, 2)
    x, g = em.Tensor(normal(rng, 60, 64)), em.Tensor(normal(rng, 60, 64))
    capi.set_deterministic(True)
    try:
        block(x, 2, 30)
        grads = [block.backward(g).to_np(), *(t.to_np() for t in block.gradients())]
        block(x, 2, 30)
        for b in (block, block.quantize8()):
            b.decode(em.Tensor(normal(rng, 6, 64)), block.make_cache(2, 10))
        for a, b in zip([block.backward(g), *block.gradients()], grads):
            np.testing.assert_array_equal(a.to_np(), b)
    finally:
        capi.set_deterministic(False)
