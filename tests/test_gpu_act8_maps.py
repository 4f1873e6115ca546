"""The BatchNorm kernels of the 8-bit activation checkpoints on maps of the size that a training step has (hundreds of partial sums, added by a launch of their own; maps
over 128 MB written past the caches), compared in float64 on the device, and their forward pass against the 32-bit unit's, bit for bit.

eps = 2^-24 is one rounding in 32 bits.  Sums over n terms of which at most 8 are added in 32 bits at a time are off by at most (8 + 4) eps times the sum of the
magnitudes (the term's own product, difference and scale: 4 roundings); each of gy's three terms carries at most 6 roundings and what the sums are off by."""
import pytest
import torch

from humaniflow_amd import _lib, act8

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def _mask(bits, M):
    """(M, C) truth values of the words' bits."""
    shift = torch.arange(32, device=bits.device, dtype=torch.int32)
    on = (bits[:, None, :] >> shift[None, :, None]) & 1
    return on.reshape(-1, bits.shape[1])[:M].bool()


@pytest.mark.parametrize('gz', [False, True])
@pytest.mark.parametrize('M,C,relu', [(18433, 256, True), (73729, 128, True), (73727, 128, False), (294900, 256, True)])
def test_bn_backward_of_large_maps(M, C, relu, gz):
    gen = torch.Generator(device='cuda').manual_seed(M + gz)
    rn = lambda *s: torch.randn(*s, generator=gen, device='cuda')
    y, g = rn(M, C) * torch.exp(0.5 * rn(C)) + rn(C), rn(M, C)
    mean, rstd = y.mean(dim=0), torch.rsqrt(y.var(dim=0, unbiased=False) + 1e-2)
    gamma, shift = rn(C), rn(C)
    y[M // 2, 5], y[M - 1, 70] = float('nan'), float('inf')                  # two markers: their channels alone are NaN
    out, ck, bits, _ = act8.bn_apply(y, gamma, shift, relu=relu)
    on = _mask(bits, M) if relu else None
    if relu:
        assert torch.equal(on, out > 0)
    del out, y
    gy, z, gg, gb = act8.bn_backward(g, ck, bits, mean, rstd, gamma, want_gz=gz)
    rz = g.double() if on is None else torch.where(on, g.double(), 0.0)
    assert z is None if not gz else torch.equal(z.double(), rz)
    del z
    xhat = (act8.unpack(ck).double() - mean.double()) * rstd.double()
    rb, rg = rz.sum(0), (rz * xhat).sum(0)
    eg, egx = 12 * EPS * rz.abs().sum(0), 12 * EPS * (rz * xhat).abs().sum(0)
    bad = torch.zeros(C, dtype=torch.bool, device='cuda')
    bad[[5, 70]] = True
    assert torch.equal(rg.isnan(), bad) and torch.equal(gg.isnan(), bad)
    assert ((gb.double() - rb).abs() <= eg).all() and ((gg.double() - rg).abs() <= egx)[~bad].all()
    ca = (gamma * rstd).double()
    want = ca * (rz - rb / M - xhat * rg / M)
    tol = ca.abs() * (8 * EPS * (rz.abs() + rb.abs() / M + (xhat * rg).abs() / M) + (eg + xhat.abs() * egx) / M)
    assert ((gy.double() - want).abs() <= tol)[:, ~bad].all() and bool(gy[:, bad].isnan().all())


@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('M,C', [(1, 64), (200, 64), (1333, 256)])
def test_forward_has_the_bits_of_the_32_bit_unit(M, C, residual, relu):
    gen = torch.Generator(device='cuda').manual_seed(M + C)
    rn = lambda *s: torch.randn(*s, generator=gen, device='cuda')
    y, scale, shift = rn(M, C) * torch.exp(2 * rn(C)), rn(C), rn(C)
    res = rn(M, C) if residual else None
    ref = torch.empty_like(y)
    _lib.check(_lib.load().hmf_bn_apply(y.data_ptr(), scale.data_ptr(), shift.data_ptr(), res.data_ptr() if residual else None, ref.data_ptr(), M, C, int(relu),
                                        _lib.current_stream()), 'hmf_bn_apply')
    assert torch.equal(act8.bn_apply(y, scale, shift, res, relu)[0], ref)
