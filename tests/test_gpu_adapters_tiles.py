"""The many-row form of the low-rank adapters in every tiling that its rule on sizes picks, against the definition in 64 bits (oracle/adapters.py, which derives what
32-bit sums may be off by; a bfloat16 result is rounded once more, by at most 2^-8 of its value).

Tiles of 128 from 192 of them on, with chunks of 64 bytes for more than 256 tiles of short bfloat16 rows; below that tiles of 64, whose reduction is split in 32 bits and,
for 4,096 elements and more, in bfloat16.  The product of the forward pass has M x N outputs and K terms, that of the backward pass M x K and N."""
import numpy as np
import pytest
import torch

from humaniflow_amd import act8, adapters
from oracle import adapters as oad

pytestmark = pytest.mark.gpu


def _case(M, K, N, r, L, kind, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    c = dict(x=rn(M, K), weight=rn(N, K) / K ** 0.5, bias=rn(N), A=rn(L, r, K) / K ** 0.5, B=rn(L, N, r) / r ** 0.5)
    c = {k: v.to(dtype).cuda() for k, v in c.items()}
    c['scale'] = (0.5 + torch.rand(L, generator=g)).cuda()
    if kind == 'runs':                                                       # in order, the first ones without an adapter
        ids = (torch.arange(M) * (L + 1) // M) - 1
    else:
        ids = torch.randint(-1, L, (M,), generator=g)
    if kind == 'past':                                                       # some ids that no adapter has
        ids[torch.randperm(M, generator=g)[:7]] = torch.tensor([L, L + 1, L, 2 ** 31 - 1, L + 9, L, L + 2])
    c['ids'] = ids.to(torch.int32).cuda()
    return c


def _d(t):
    return t.detach().double().cpu().numpy()


def _host(c):
    return [_d(c[k]) for k in ('weight', 'A', 'B', 'scale')] + [c['ids'].cpu().numpy()]


def _near(got, ref, bound):
    tol = bound + (2.0 ** -8 * np.abs(ref) if got.dtype == torch.bfloat16 else 0.0) + 1e-37
    got = _d(got)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = np.isnan(ref) | (np.abs(got - ref) <= tol)
    assert ok.all(), (np.abs(got - ref)[~ok].max(), np.argwhere(~ok)[:4].tolist(), int((~ok).sum()))


F32, B16 = torch.float32, torch.bfloat16
#          M     K     N     r   L    kind      what it picks
FORWARD = [(F32, 1700, 520, 1800, 16, 5, 'mixed'),     # 14 x 15 tiles of 128, chunks of 128 bytes
           (F32, 2300, 130, 2001, 3, 300, 'runs'),     # 18 x 16; some twenty adapters a tile
           (B16, 1700, 1000, 1800, 16, 40, 'mixed'),   # 14 x 15
           (B16, 1701, 1100, 2300, 33, 9, 'past'),     # 14 x 18, longer rows: chunks of 128 bytes
           (B16, 2300, 1000, 2000, 16, 5, 'mixed'),    # 18 x 16 tiles of short rows: chunks of 64 bytes
           (B16, 2299, 72, 2050, 7, 300, 'past'),      # 18 x 17, one chunk of the ring's four stages
           (B16, 300, 4100, 70, 8, 6, 'mixed'),        # tiles of 64, two splits in bfloat16
           (F32, 300, 1100, 70, 8, 6, 'past')]         # tiles of 64, splits in 32 bits
BACKWARD = [(F32, 1700, 1800, 520, 16, 5, 'mixed'), (F32, 2300, 2001, 130, 3, 300, 'runs'), (B16, 1700, 1800, 1000, 16, 40, 'past'), (B16, 1701, 2300, 1100, 33, 9, 'mixed'),
            (B16, 2300, 2000, 1000, 16, 5, 'mixed'), (B16, 2299, 2050, 72, 7, 300, 'runs'), (B16, 300, 70, 4100, 8, 6, 'mixed')]


@pytest.mark.parametrize('dtype,M,K,N,r,L,kind', FORWARD)
def test_forward_in_every_tiling(dtype, M, K, N, r, L, kind):
    c = _case(M, K, N, r, L, kind, dtype, M + K + N)
    y, t = adapters.adapted_linear_forward(**c)
    w, a, b, scale, ids = _host(c)
    ry, rt, ey, et = oad.forward(_d(c['x']), w, _d(c['bias']), a, b, scale, ids)
    _near(y, ry, ey)
    _near(t, rt, et)


@pytest.mark.parametrize('x8', [False, True])
@pytest.mark.parametrize('dtype,M,K,N,r,L,kind', BACKWARD)
def test_backward_in_every_tiling(dtype, M, K, N, r, L, kind, x8):
    c = _case(M, K, N, r, L, kind, dtype, M + K + N)
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    t = adapters.adapted_linear_forward(**c)[1]
    x = act8.pack(c['x']) if x8 else c['x']
    got = adapters.adapted_linear_backward(dy, x, t, c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    known = (c['ids'] < L).cpu().numpy()                                     # a row whose id no adapter has has t = NaN and is in no gradient
    t = np.where(known[:, None], _d(t), 0.0)
    rx, ra, rb, ex, ea, eb = oad.backward(_d(dy), _d(act8.unpack(x)) if x8 else _d(c['x']), t, *_host(c))
    for g, ref, bound in zip(got, (rx, ra, rb), (ex, ea, eb)):
        _near(g, ref, bound)


@pytest.mark.parametrize('dtype,M,K,N', [(F32, 1700, 520, 1800), (B16, 1700, 520, 1800), (B16, 2300, 520, 2000)])
def test_infinities_stay_with_their_adapter_in_tiles_of_128(dtype, M, K, N):
    """Infinite and NaN weights of one adapter, in rows and columns of a tile that other adapters share: the others' results keep their bits, forward and backward."""
    L = 40
    c = _case(M, K, N, 6, L, 'mixed', dtype, 3)
    args = lambda: (c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    y0, t = adapters.adapted_linear_forward(**c)
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    back = lambda: adapters.adapted_linear_backward(dy, c['x'], t, *args())
    x0, a0, b0 = back()
    c['B'][7, 130, 1], c['B'][7, 1, 0], c['A'][7, 0, 200] = float('nan'), float('inf'), float('-inf')
    y, _ = adapters.adapted_linear_forward(**c)
    dx, dA, dB = back()
    other, rest = c['ids'] != 7, torch.arange(L, device='cuda') != 7
    assert torch.equal(y[other], y0[other]) and torch.equal(dx[other], x0[other])
    assert torch.equal(dA[rest], a0[rest]) and torch.equal(dB[rest], b0[rest])
    mine = ~other
    assert bool(mine.any()) and not torch.isfinite(y[mine][:, [1, 130]]).any() and not torch.isfinite(dx[mine][:, 200]).any()
