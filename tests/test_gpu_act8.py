"""8-bit activation checkpoints on the device against the definitions in 64 bits (oracle/act8.py), and the encoder's training graph that keeps them.

Tolerances: eps = 2^-24 is one rounding in 32 bits.  Codes, exponents and bits are whole numbers and have to be equal.  Sums over n terms of which at most 8 are
added in 32 bits at a time are off by at most (8 + 4) eps times the sum of the magnitudes (the term's own product, difference and scale: 4 roundings)."""
import copy

import numpy as np
import pytest
import torch

from humaniflow_amd import act8
from humaniflow_amd import encoder_train as et
from humaniflow_amd.encoder import ResNetEncoder
from oracle import act8 as oact

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def _rows(M, C, seed, pad=0, dtype=torch.float32, spread=4.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, C + pad, generator=g) * torch.exp(spread * torch.randn(C + pad, generator=g))
    return x.to(dtype).cuda()[:, :C]


def _same(ck, x):
    codes, exps = oact.pack(x.double().cpu().numpy())
    assert np.array_equal(ck.codes.cpu().numpy(), codes)
    assert np.array_equal(ck.exps.cpu().numpy().astype(np.int64) - 133, exps)
    return codes, exps


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,C,pad', [(1, 1, 0), (1, 64, 0), (31, 64, 0), (32, 128, 0), (33, 128, 8), (65, 130, 3), (7, 515, 13), (100, 257, 0), (64, 8, 0),
                                     (97, 200, 56), (300, 72, 1)])
def test_pack_and_unpack(M, C, pad, dtype):
    x = _rows(M, C, M + C, pad, dtype)
    ck = act8.pack(x)
    codes, exps = _same(ck, x)
    v = oact.values(codes, exps)
    for dt in (torch.float32, torch.bfloat16):
        got = act8.unpack(ck, dt)
        assert got.dtype == dt and np.array_equal(got.double().cpu().numpy(), v)


def test_pack_extremes():
    """Zeros, denormals, the largest finite values, a magnitude that would round to 128 steps, ties, infinities and NaN."""
    big = float(np.finfo(np.float32).max)
    col = lambda *v: list(v) + [0.0] * (32 - len(v))
    cols = [col(0.0), col(1e-45, -3e-39, 1e-38), col(big, -big, 1.0), col(127.5 / 64, 1.0), col(127.4999 / 64, 1.0), col(64.0, 0.5, 1.5, 2.5, -0.5, -1.5),
            col(float('inf'), 2.0, -1.0), col(float('nan'), float('-inf')), col(float('nan'), 1e-30)]
    x = torch.tensor(cols, dtype=torch.float32).t().contiguous().cuda()
    for t in (x, torch.cat([x, x[:5]]), torch.cat([x, x], dim=1)[:, :16]):
        ck = act8.pack(t)
        codes, exps = _same(ck, t)
        assert np.array_equal(act8.unpack(ck).double().cpu().numpy(), oact.values(codes, exps), equal_nan=True)


def test_pack_of_views_and_empty_rows():
    wide = _rows(40, 96, 0)
    for x in (wide[:, 1:65], wide[::3, :64], wide.t(), wide[:, ::2], wide[5:6], wide[:1].expand(33, 96), wide[:, 7:8]):
        _same(act8.pack(x), x)
    for shape in ((0, 64), (5, 0)):
        e = act8.pack(torch.empty(shape, device='cuda'))
        assert tuple(act8.unpack(e).shape) == shape


def test_pack_beyond_32_bit_offsets():
    """More than 2^31 elements: the last rows are where an offset that wrapped would show."""
    M, C = 1049000, 2048
    x = torch.zeros(M, C, dtype=torch.bfloat16, device='cuda')
    tail = _rows(1000, C, 3, dtype=torch.bfloat16, spread=1.0)
    x[-1000:] = tail
    ck = act8.pack(x)
    ref = tail[-(192 + M % 32):]                                             # whole blocks at the end
    codes, exps = oact.pack(ref.double().cpu().numpy())
    n = ref.shape[0]
    assert np.array_equal(ck.codes[-n:].cpu().numpy(), codes)
    y = act8.unpack(ck, torch.bfloat16)
    assert np.array_equal(y[-n:].double().cpu().numpy(), oact.values(codes, exps)) and not bool(y[:1000].any())


def _bn_case(M, C, seed, residual):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(M, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + torch.randn(C, generator=g)
    scale, shift = torch.randn(C, generator=g), torch.randn(C, generator=g)
    res = torch.randn(M, C, generator=g).cuda() if residual else None
    return y.cuda(), scale.cuda(), shift.cuda(), res


@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('M,C', [(1, 64), (31, 64), (32, 192), (75, 128), (1000, 64), (130, 512)])
def test_bn_apply_and_restore(M, C, relu, residual):
    y, scale, shift, res = _bn_case(M, C, M + C, residual)
    out, ck, bits, ck_out = act8.bn_apply(y, scale, shift, res, relu, keep_out=True)
    codes, exps = _same(ck, y)
    a = y.double() * scale.double() + shift.double()
    v = a + (res.double() if residual else 0.0)
    ref = v.clamp(min=0) if relu else v
    assert bool(((out.double() - ref).abs() <= EPS * (a.abs() + v.abs()) * 1.001).all())
    _same(ck_out, out)
    if relu:
        assert np.array_equal(oact.mask_of(bits.cpu().numpy().view(np.uint32), M), (out > 0).cpu().numpy())
    else:
        assert bits is None
    again, _, _, none = act8.bn_apply(y, scale, shift, res, relu)
    assert none is None and torch.equal(again, out)
    x = act8.restore_activation(ck, scale, shift, bits)
    w = oact.values(codes, exps) * scale.double().cpu().numpy() + shift.double().cpu().numpy()
    w = torch.from_numpy(w).cuda()
    if relu:
        w = torch.where(out > 0, w.clamp(min=0), torch.zeros_like(w))
    if relu and residual:
        return                                                               # not how an identity unit is rebuilt: its out has a checkpoint of its own
    assert bool(((x.double() - w).abs() <= EPS * w.abs() * 1.001).all())


def test_bn_apply_matches_the_32_bit_unit_and_keeps_nan():
    from humaniflow_amd import _lib
    y, scale, shift, res = _bn_case(200, 64, 5, True)
    ref = torch.empty_like(y)
    _lib.check(_lib.load().hmf_bn_apply(y.data_ptr(), scale.data_ptr(), shift.data_ptr(), res.data_ptr(), ref.data_ptr(), 200, 64, 1, _lib.current_stream()))
    out = act8.bn_apply(y, scale, shift, res)[0]
    assert bool(((out - ref).abs() <= 2 * EPS * (ref.abs() + res.abs() + 1)).all())
    y[3, 5], y[40, 6] = float('nan'), float('inf')
    out, ck, bits, ck_out = act8.bn_apply(y, scale.abs(), shift, None, keep_out=True)
    assert torch.isnan(out[3, 5]) and torch.isinf(out[40, 6])
    x = act8.restore_activation(ck, scale.abs(), shift, bits)
    assert torch.isnan(x[3, 5]) and torch.isnan(x[40, 6]) and int(torch.isnan(x).sum()) == 2
    assert int(torch.isnan(act8.unpack(ck_out)).sum()) == 2


@pytest.mark.parametrize('gz', [False, True])
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('M,C', [(1, 64), (33, 64), (75, 128), (4608, 64), (700, 512), (20011, 64)])
def test_bn_backward(M, C, masked, gz):
    y, scale, shift, _ = _bn_case(M, C, 3 * M + C, False)
    g = torch.randn(M, C, generator=torch.Generator().manual_seed(M)).cuda()
    mean = y.mean(dim=0)
    rstd = torch.rsqrt(y.var(dim=0, unbiased=False) + 1e-2)
    gamma = scale
    _, ck, bits, _ = act8.bn_apply(y, scale, shift, relu=masked)
    gy, z, gg, gb = act8.bn_backward(g, ck, bits, mean, rstd, gamma, want_gz=gz)
    d = lambda t: t.double().cpu().numpy()
    yq = d(act8.unpack(ck))
    xhat = (yq - d(mean)) * d(rstd)
    mask = oact.mask_of(bits.cpu().numpy().view(np.uint32), M) if masked else np.ones((M, C), bool)
    rz, rg, rb, ry = oact.bn_backward(d(g), xhat, mask, d(rstd), d(gamma))
    if gz:
        assert np.array_equal(d(z), rz)
    else:
        assert z is None
    mz, mzx = np.abs(rz).sum(axis=0), np.abs(rz * xhat).sum(axis=0)
    eg, egx = 12 * EPS * mz, 12 * EPS * mzx
    assert np.all(np.abs(d(gb) - rb) <= eg + 1e-300) and np.all(np.abs(d(gg) - rg) <= egx + 1e-300)
    ca = np.abs(d(gamma) * d(rstd))
    # gy: each of its three terms carries at most 6 roundings, and the two means what the sums are off by
    tol = ca * (8 * EPS * (np.abs(rz) + np.abs(rb) / M + np.abs(xhat * rg) / M) + (eg + np.abs(xhat) * egx) / M)
    assert np.all(np.abs(d(gy) - ry) <= tol + 1e-300)
    again = act8.bn_backward(g, ck, bits, mean, rstd, gamma, want_gz=gz)
    assert torch.equal(again[0], gy) and torch.equal(again[2], gg) and torch.equal(again[3], gb)      # no atomics: bit for bit


@pytest.mark.parametrize('gz', [False, True])
def test_bn_backward_of_few_rows_and_many_channels(gz):
    """A map over 128 MB whose partial sums are few: 256 rows of 131,136 channels.  Compared in float64 on the device, tolerances as above."""
    M, C = 256, 131136
    gen = torch.Generator(device='cuda').manual_seed(5)
    y = torch.randn(M, C, generator=gen, device='cuda')
    g = torch.randn(M, C, generator=gen, device='cuda')
    mean = y.mean(dim=0)
    rstd = torch.rsqrt(y.var(dim=0, unbiased=False) + 1e-2)
    gamma = 0.5 + torch.rand(C, generator=gen, device='cuda')
    ck = act8.pack(y)
    got = act8.bn_backward(g, ck, None, mean, rstd, gamma, want_gz=gz)
    assert not gz or torch.equal(got[1], g)
    xhat = (act8.unpack(ck).double() - mean.double()) * rstd.double()
    z = g.double()
    gb, gg = z.sum(0), (z * xhat).sum(0)
    eg, egx = 12 * EPS * z.abs().sum(0), 12 * EPS * (z * xhat).abs().sum(0)
    assert ((got[3].double() - gb).abs() <= eg).all() and ((got[2].double() - gg).abs() <= egx).all()
    ca = (gamma * rstd).double()
    tol = ca * (8 * EPS * (z.abs() + gb.abs() / M + (xhat * gg).abs() / M) + (eg + xhat.abs() * egx) / M)
    assert ((got[0].double() - ca * (z - gb / M - xhat * gg / M)).abs() <= tol).all()


def test_refusals_on_the_device():
    y, scale, shift, res = _bn_case(64, 64, 0, True)
    ck = act8.pack(y)
    with pytest.raises(ValueError, match='64 channels'):
        act8.bn_apply(y[:, :32].contiguous(), scale[:32], shift[:32])
    with pytest.raises(ValueError, match='residual'):
        act8.bn_apply(y, scale, shift, res[:32])
    with pytest.raises(ValueError, match='contiguous'):
        act8.bn_apply(y.t(), scale, shift)
    with pytest.raises(ValueError, match='checkpoint holds'):
        act8.bn_backward(res[:32].contiguous(), ck, None, scale, scale, scale)
    with pytest.raises(ValueError, match='bits'):
        act8.bn_backward(res, ck, torch.zeros(1, 64, dtype=torch.int32, device='cuda'), scale, scale, scale)
    with pytest.raises(ValueError, match='is on cpu'):
        act8.bn_backward(res, ck, None, scale.cpu(), scale, scale)
    with pytest.raises(RuntimeError, match='aligned'):
        act8.bn_apply(torch.randn(64 * 64 + 1, device='cuda')[1:].view(64, 64), scale, shift)
    with pytest.raises(ValueError, match='float32 or bfloat16'):
        act8.pack(y.half())


def test_own_stream_and_graph_replays():
    y, scale, shift, res = _bn_case(1000, 128, 9, True)
    g = torch.randn(1000, 128, device='cuda')
    mean, rstd = y.mean(dim=0), torch.rsqrt(y.var(dim=0) + 1e-3)

    def step():
        out, ck, bits, ck_out = act8.bn_apply(y, scale, shift, res, keep_out=True)
        return [out, act8.unpack(ck_out), *act8.bn_backward(g, ck, bits, mean, rstd, scale, want_gz=True)]
    ref = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        y.mul_(1.5)
        g.add_(0.25)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), k


# ---- the encoder's training graph ---------------------------------------------------------------------------------------------
def _grads(enc, x, w):
    for p in enc.parameters():
        p.grad = None
    f = enc(x)
    (f * w).sum().backward()
    return f.detach().clone(), {n: p.grad.clone() for n, p in enc.named_parameters()}


@pytest.mark.parametrize('layers,fused_stem', [(18, True), (50, True), (18, False)])
def test_encoder_training_with_int8_checkpoints(layers, fused_stem, monkeypatch):
    """Forward values as without checkpoints (one more rounding where an identity is added); gradients within the checkpoints' rounding of the 32-bit ones.
    A kept value is off by a uniform error of at most step / 2, step <= 2 amax / 127: relative to the root mean square of a block of 32 normal values (amax about
    2.1 rms) 2 * 2.1 / 127 / sqrt(12) = 0.95 % at most.  The gradient of a layer is linear in that error where the layer's own x and xhat enter, and the errors of
    the layers above come down through gy alone (xhat's share of it): below 5 % of the gradient's norm for each parameter, and 1.5 % over all of them."""
    monkeypatch.setattr(et, 'STEM_TAIL_FUSED', fused_stem)
    torch.manual_seed(layers)
    enc = ResNetEncoder(layers, 18).cuda().train()
    ref = copy.deepcopy(enc)
    x = torch.randn(8, 18, 128, 128, device='cuda')
    w = torch.randn(8, 512 if layers == 18 else 2048, device='cuda')
    fr, gr = _grads(ref, x, w)
    enc.activation_checkpoint = 'int8'
    fe, ge = _grads(enc, x, w)
    assert ((fe - fr).norm() / fr.norm()).item() < 1e-5
    for a, b in zip(enc.buffers(), ref.buffers()):
        assert torch.allclose(a.float(), b.float(), rtol=1e-5, atol=1e-6)
    num = den = 0.0
    for n in gr:
        d, m = (ge[n].double() - gr[n].double()).norm().item(), gr[n].double().norm().item()
        assert d <= 0.05 * m, (n, d / m)
        num, den = num + d * d, den + m * m
    assert (num / den) ** 0.5 < 0.015


def test_encoder_checkpoints_hold_less_memory_and_free_it():
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    x = torch.randn(16, 18, 256, 256, device='cuda')
    held = {}
    for mode in (None, 'int8'):
        enc.activation_checkpoint = mode
        enc(x).sum().backward()                                               # warm: packs and buffers that stay
        for p in enc.parameters():
            p.grad = None
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        f = enc(x)
        held[mode] = torch.cuda.memory_allocated() - base
        f.sum().backward()
        with pytest.raises(RuntimeError, match='already back-propagated'):
            f.grad_fn.apply(torch.ones_like(f))
        for p in enc.parameters():
            p.grad = None
        del f
    assert held['int8'] < 0.4 * held[None], held


def test_encoder_refuses_an_unknown_checkpoint():
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.activation_checkpoint = 'fp8'
    with pytest.raises(ValueError, match='activation_checkpoint'):
        enc(torch.randn(1, 18, 64, 64, device='cuda'))


def test_captured_training_pass_with_int8_checkpoints():
    """Forward and backward of the encoder in one graph, replayed with other inputs and the program's own work between; the weight gradients' sums use float atomics, so
    they are compared within 1e-4 of their norm."""
    torch.manual_seed(1)
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.activation_checkpoint = 'int8'
    x, w = torch.randn(4, 18, 64, 64, device='cuda'), torch.randn(4, 512, device='cuda')

    def step():
        f = enc(x)
        return (f, *torch.autograd.grad((f * w).sum(), list(enc.parameters())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        w.mul_(0.7)
        graph.replay()
        got = [t.detach().clone() for t in held]
        want = [t.detach() for t in step()]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert (a - b).norm().item() <= 1e-4 * b.norm().item() + 1e-12, k
