"""Low-rank adapters and BatchNorm checkpoints at the ends of the sizes: one row, column and rank, and tensors of more than 2^31 elements.  Bounds as in oracle/adapters.py."""
import numpy as np
import pytest
import torch

from humaniflow_amd import act8, adapters
from oracle import adapters as oad

pytestmark = pytest.mark.gpu


def _d(t):
    return t.detach().double().cpu().numpy()


def _near(got, ref, bound):
    tol = bound + (2.0 ** -8 * np.abs(ref) if got.dtype == torch.bfloat16 else 0.0) + 1e-37
    assert (np.abs(_d(got) - ref) <= tol).all()


def _params(K, N, r, L, dtype, g):
    rn = lambda *s: torch.randn(*s, generator=g)
    p = dict(weight=rn(N, K) / K ** 0.5, bias=rn(N), A=rn(L, r, K) / K ** 0.5, B=rn(L, N, r) / r ** 0.5)
    return {**{k: v.to(dtype).cuda() for k, v in p.items()}, 'scale': (0.5 + torch.rand(L, generator=g)).cuda()}


def _host(p, ids):
    return [_d(p[k]) for k in ('weight', 'A', 'B', 'scale')] + [ids.cpu().numpy()]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,r,L', [(1, 1, 1, 1, 1), (4, 3, 2, 64, 1), (5, 1, 1, 1, 1), (256, 3, 2, 64, 256), (300, 1, 1, 1, 1), (300, 1, 200, 64, 2), (257, 70, 1, 64, 300),
                                       (1000, 2, 3, 1, 1)])
def test_smallest_sizes(M, K, N, r, L, dtype):
    g = torch.Generator().manual_seed(M + K)
    p, x, dy = _params(K, N, r, L, dtype, g), torch.randn(M, K, generator=g).to(dtype).cuda(), torch.randn(M, N, generator=g).to(dtype).cuda()
    ids = torch.randint(-1, L, (M,), generator=g).to(torch.int32).cuda()
    y, t = adapters.adapted_linear_forward(x, ids=ids, **p)
    w, a, b, scale, hid = _host(p, ids)
    ry, rt, ey, et = oad.forward(_d(x), w, _d(p['bias']), a, b, scale, hid)
    _near(y, ry, ey)
    _near(t, rt, et)
    del p['bias']
    for kept in (x, act8.pack(x)):
        got = adapters.adapted_linear_backward(dy, kept, t, ids=ids, **p)
        rx, ra, rb, ex, ea, eb = oad.backward(_d(dy), _d(x) if kept is x else _d(act8.unpack(kept)), _d(t), w, a, b, scale, hid)
        for v, ref, bound in zip(got, (rx, ra, rb), (ex, ea, eb)):
            _near(v, ref, bound)


@pytest.mark.parametrize('K', [1024, 1030])
def test_rows_past_32_bit_offsets(K):
    """2.2 million rows of 1,024 (and of 1,030, which are copied into whole chunks): all but the last 900 are zero, so that the gradients are theirs alone."""
    M, N, r, L, n = 2200000, 8, 4, 3, 900
    g = torch.Generator().manual_seed(K)
    p = _params(K, N, r, L, torch.bfloat16, g)
    tail, dtail = torch.randn(n, K, generator=g).bfloat16().cuda(), torch.randn(n, N, generator=g).bfloat16().cuda()
    x, dy = torch.zeros(M, K, dtype=torch.bfloat16, device='cuda'), torch.zeros(M, N, dtype=torch.bfloat16, device='cuda')
    x[-n:], dy[-n:] = tail, dtail
    assert M * K > 2 ** 31
    ids = (torch.arange(M, device='cuda') % 4 - 1).to(torch.int32)
    y, t = adapters.adapted_linear_forward(x, ids=ids, **p)
    w, a, b, scale, hid = _host(p, ids[-n:])
    ry, rt, ey, et = oad.forward(_d(tail), w, _d(p['bias']), a, b, scale, hid)
    _near(y[-n:], ry, ey)
    _near(t[-n:], rt, et)
    assert bool((y[:-n] == p.pop('bias')).all()) and not bool(t[:-n].any())
    rx, ra, rb, ex, ea, eb = oad.backward(_d(dtail), _d(tail), _d(t[-n:]), w, a, b, scale, hid)
    dx, dA, dB = adapters.adapted_linear_backward(dy, x, t, ids=ids, **p)
    _near(dx[-n:], rx, ex)
    _near(dA, ra, ea)
    _near(dB, rb, eb)
    assert not bool(dx[:-n].any())


@pytest.mark.parametrize('M', [3, 40, 300])
def test_adapters_past_32_bit_offsets(M):
    """A of 60,000 adapters x 16 x 2,304: the last ones lie behind 2^31 elements; the gradients of those without rows are zeros."""
    K, N, r, L, n = 2304, 8, 16, 60000, 5
    g = torch.Generator().manual_seed(M)
    p = _params(K, N, r, n, torch.bfloat16, g)
    A, B = torch.zeros(L, r, K, dtype=torch.bfloat16, device='cuda'), torch.zeros(L, N, r, dtype=torch.bfloat16, device='cuda')
    A[-n:], B[-n:] = p['A'], p['B']
    scale = torch.ones(L, device='cuda')
    scale[-n:] = p['scale']
    assert (L - n) * r * K > 2 ** 31
    x, dy = torch.randn(M, K, generator=g).bfloat16().cuda(), torch.randn(M, N, generator=g).bfloat16().cuda()
    low = torch.randint(-1, n, (M,), generator=g)
    ids = torch.where(low < 0, low, low + L - n).to(torch.int32).cuda()
    y, t = adapters.adapted_linear_forward(x, p['weight'], p['bias'], A, B, scale, ids)
    w, a, b, s, hid = _host(p, low)
    ry, rt, ey, et = oad.forward(_d(x), w, _d(p['bias']), a, b, s, hid)
    _near(y, ry, ey)
    _near(t, rt, et)
    dx, dA, dB = adapters.adapted_linear_backward(dy, x, t, p['weight'], A, B, scale, ids)
    rx, ra, rb, ex, ea, eb = oad.backward(_d(dy), _d(x), _d(t), w, a, b, s, hid)
    _near(dx, rx, ex)
    _near(dA[-n:], ra, ea)
    _near(dB[-n:], rb, eb)
    assert not bool(dA[:-n].any()) and not bool(dB[:-n].any())


def test_a_unit_past_32_bit_offsets():
    """BatchNorm with its checkpoints and its backward pass on 4.4 million rows of 512: the last 64 blocks are those of a map of their own, and with a gradient in them alone
    they are what gy, d gamma and d beta have (tolerances as in test_gpu_act8.py)."""
    M, C, n, eps = 4400000, 512, 64 * 32, 2.0 ** -24
    assert M % 32 == 0 and M * C > 2 ** 31
    gen = torch.Generator(device='cuda').manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device='cuda')
    y, scale, shift, tail, gt = torch.zeros(M, C, device='cuda'), rn(C), rn(C), rn(n, C), rn(n, C)
    y[-n:] = tail
    out, ck, bits, ck_out = act8.bn_apply(y, scale, shift, relu=True, keep_out=True)
    ref, rk, rbits, rk_out = act8.bn_apply(tail, scale, shift, relu=True, keep_out=True)
    assert torch.equal(out[-n:], ref) and torch.equal(bits[-n // 32:], rbits)
    for p, q in ((ck, rk), (ck_out, rk_out)):
        assert torch.equal(p.codes[-n:], q.codes) and torch.equal(p.exps[-n // 32:], q.exps)
    del out, y
    assert torch.equal(act8.restore_activation(ck, scale, shift, bits)[-n:], act8.restore_activation(rk, scale, shift, rbits))
    g = torch.zeros(M, C, device='cuda')
    g[-n:] = gt
    mean, rstd, gamma = tail.mean(0), torch.rsqrt(tail.var(0) + 1e-2), scale
    gy, _, gg, gb = act8.bn_backward(g, ck, bits, mean, rstd, gamma)
    z = torch.where(ref > 0, gt.double(), 0.0)
    xhat = (act8.unpack(rk).double() - mean.double()) * rstd.double()
    rb, rg = z.sum(0), (z * xhat).sum(0)
    eg, egx = 12 * eps * z.abs().sum(0), 12 * eps * (z * xhat).abs().sum(0)
    assert ((gb.double() - rb).abs() <= eg).all() and ((gg.double() - rg).abs() <= egx).all()
    ca = (gamma * rstd).double()
    want = ca * (z - rb / M - xhat * rg / M)
    tol = ca.abs() * (8 * eps * (z.abs() + rb.abs() / M + (xhat * rg).abs() / M) + (eg + xhat.abs() * egx) / M)
    assert ((gy[-n:].double() - want).abs() <= tol).all()
    first = -ca * (rb / M - mean.double() * rstd.double() * rg / M)          # a row of zeros: xhat = -mean rstd
    tol = ca.abs() * (8 * eps * (rb.abs() / M + (mean * rstd * rg).abs().double() / M) + (eg + (mean * rstd).abs() * egx) / M)
    assert ((gy[:n].double() - first).abs() <= tol).all()
