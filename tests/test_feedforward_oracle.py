"""The oracle of RMS norm, 8-bit matrices and gated layers: against closed forms
and finite differences.  CPU only."""

import numpy as np
import pytest

from oracle import feedforward as ff


def test_e4m3_sizes():
    assert len(ff.E4M3) == 127 and ff.E4M3[126] == 448 and ff.E4M3[1] == 2.0 ** -9 and ff.E4M3[8] == 2.0 ** -6 and ff.E4M3[0x38] == 1
    assert (np.diff(ff.E4M3) > 0).all()


def test_e4m3_is_torchs():
    torch = pytest.importorskip("torch")
    x = torch.randn(4096, generator=torch.Generator().manual_seed(1)) * torch.exp(3 * torch.randn(4096, generator=torch.Generator().manual_seed(2)))
    x = x.clamp(-448, 448)
    codes, scales = ff.quantise8(np.pad(x.numpy().reshape(-1, 64), ((0, 0), (0, 64)), constant_values=448))
    assert (scales[:, 0] == 127).all()  # 448 in every group: the scale is 1
    np.testing.assert_array_equal(codes[:, :64].reshape(-1), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_scale_is_the_least_that_cuts_nothing():
    for amax, byte in ((448, 127), (np.nextafter(np.float32(448), np.float32(1e9)), 128), (1.75, 119), (1.7500001, 120), (2 ** -111, 8),
                       (2.0 ** -149, 8), (0, 127), (np.nan, 255), (np.inf, 255), (2.0 ** 127, 255), (np.nextafter(np.float32(2.0 ** 127), np.float32(0)), 246)):
        x = np.zeros((1, 130), np.float32)
        x[0, 5] = -amax if amax == amax else amax
        codes, scales = ff.quantise8(x)
        assert scales.tolist() == [[byte, 127, 127, 127]], amax
        assert (codes[0, 128:] == 0).all()


def test_rounding_is_within_half_a_step_and_ties_go_to_even():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((7, 300)) * np.exp(2 * rng.standard_normal((7, 300)))).astype(np.float32)
    v = ff.values8(*ff.quantise8(x), 300)
    step = np.repeat(2.0 ** (ff.quantise8(x)[1].astype(float) - 127), 128, 1)[:, :300]
    assert (np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * step)).all()
    x = np.full((1, 128), 448, np.float32)
    x[0, :4] = 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10  # between 1 and 1.125, 1.125 and 1.25, 0 and 2^-9, 2^-9 and 2^-8
    assert ff.values8(*ff.quantise8(x), 4).tolist() == [[1, 1.25, 0, 2.0 ** -8]]


def _difference(f, x, at, h=1e-6):
    up, down = x.copy(), x.copy()
    up[at] += h
    down[at] -= h
    return (f(up) - f(down)) / (2 * h)


def test_rmsnorm_gradient_by_differences():
    rng = np.random.default_rng(5)
    s, gamma, dy = rng.standard_normal((3, 8)), rng.standard_normal(8), rng.standard_normal((3, 8))
    _, rstd = ff.rmsnorm_fwd(s, gamma, 0.01)
    dx, dgamma = ff.rmsnorm_bwd(s, gamma, rstd, dy)
    for at in np.ndindex(3, 8):
        assert abs(_difference(lambda v: (ff.rmsnorm_fwd(v, gamma, 0.01)[0] * dy).sum(), s, at) - dx[at]) < 1e-7
    for j in range(8):
        assert abs(_difference(lambda v: (ff.rmsnorm_fwd(s, v, 0.01)[0] * dy).sum(), gamma, (j,)) - dgamma[j]) < 1e-7


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gate_gradient_by_differences(act):
    rng = np.random.default_rng(6)
    pre, dh = 3 * rng.standard_normal((4, 10)), rng.standard_normal((4, 5))
    grad = ff.gate_bwd(act, dh, pre)
    for at in np.ndindex(4, 10):
        assert abs(_difference(lambda v: (ff.gate(act, v) * dh).sum(), pre, at) - grad[at]) < 1e-7
