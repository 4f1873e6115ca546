"""The low-rank adapters in exactly the workspace that the size query names, with a guard behind it, and what a call holds of the card."""
import numpy as np
import pytest
import torch

from humaniflow_amd import _lib, adapters
from oracle import adapters as oad

pytestmark = pytest.mark.gpu


def _d(t):
    return t.detach().double().cpu().numpy()


def _near(got, ref, bound):
    tol = bound + (2.0 ** -8 * np.abs(ref) if got.dtype == torch.bfloat16 else 0.0) + 1e-37
    assert (np.abs(_d(got) - ref) <= tol).all()


def _case(counts, none, K, N, r, dtype):
    """Adapter l has counts[l] rows, `none` rows have none, in random order."""
    g = torch.Generator().manual_seed(len(counts))
    ids = torch.cat([torch.full((n,), l) for l, n in enumerate(counts)] + [torch.full((none,), -1)])
    ids = ids[torch.randperm(len(ids), generator=g)]
    M, L = len(ids), len(counts)
    rn = lambda *s: torch.randn(*s, generator=g)
    c = dict(x=rn(M, K), weight=rn(N, K) / K ** 0.5, bias=rn(N), A=rn(L, r, K) / K ** 0.5, B=rn(L, N, r) / r ** 0.5)
    c = {k: v.to(dtype).cuda() for k, v in c.items()}
    c['scale'], c['ids'] = (0.5 + torch.rand(L, generator=g)).cuda(), ids.to(torch.int32).cuda()
    return c


def _guarded(n):
    ws = torch.full((n + 4096,), 0xa5, dtype=torch.uint8, device='cuda')
    return ws, lambda: bool((ws[n:] == 0xa5).all())


COUNTS = [[600] + [3] * 69 + [256] + [1] * 9 + [257] + [0] * 30 + [300, 0, 512, 2],      # several pieces in three different groups of 64 adapters
          [1] * 70 + [258] + [0] * 60 + [2] + [259], [300], [256] * 3, [7, 5]]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('K,N', [(128, 192), (130, 75)])
@pytest.mark.parametrize('counts', COUNTS, ids=[str(k) for k in range(len(COUNTS))])
def test_results_in_the_named_workspace(counts, K, N, dtype):
    lib, r, bf16 = _lib.load(), 5, int(dtype == torch.bfloat16)
    c = _case(counts, 40, K, N, r, dtype)
    M, L, st = c['x'].shape[0], len(counts), _lib.current_stream()
    p = {k: v.data_ptr() for k, v in c.items()}
    y, t = torch.empty(M, N, dtype=dtype, device='cuda'), torch.empty(M, r, device='cuda')
    n = lib.hmf_adapted_linear_workspace_bytes_for(p['x'], K, p['weight'], p['A'], M, K, N, r, L, bf16)
    ws, whole = _guarded(n)
    _lib.check(lib.hmf_adapted_linear(p['x'], K, p['weight'], p['bias'], p['A'], p['B'], p['scale'], p['ids'], M, K, N, r, L, bf16, y.data_ptr(), t.data_ptr(),
                                      ws.data_ptr(), n, st))
    host = [_d(c[k]) for k in ('weight', 'A', 'B', 'scale')] + [c['ids'].cpu().numpy()]
    ry, rt, ey, et = oad.forward(_d(c['x']), host[0], _d(c['bias']), *host[1:])
    _near(y, ry, ey)
    _near(t, rt, et)
    assert whole()
    dy = torch.randn(M, N, device='cuda').to(dtype)
    rx, ra, rb, ex, ea, eb = oad.backward(_d(dy), _d(c['x']), _d(t), *host)
    for need_dx in (1, 0):
        dx, dA, dB = torch.empty_like(c['x']), torch.empty_like(c['A']), torch.empty_like(c['B'])
        n = lib.hmf_adapted_linear_backward_workspace_bytes_for(M, K, N, r, L, bf16, need_dx)
        ws, whole = _guarded(n)
        _lib.check(lib.hmf_adapted_linear_backward(dy.data_ptr(), p['x'], K, None, t.data_ptr(), p['weight'], p['A'], p['B'], p['scale'], p['ids'], M, K, N, r, L, bf16,
                                                   dx.data_ptr() if need_dx else None, dA.data_ptr(), dB.data_ptr(), ws.data_ptr(), n, st))
        if need_dx:
            _near(dx, rx, ex)
        _near(dA, ra, ea)
        _near(dB, rb, eb)
        assert whole()


def test_many_adapters_do_not_cost_memory():
    """4,096 rows and 2,000 adapters, 1,024 -> 512, rank 32: beside its results the forward holds t and the plan, the backward the two transposed operands and little more."""
    g = torch.Generator(device='cuda').manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, device='cuda').bfloat16()
    M, K, N, r, L = 4096, 1024, 512, 32, 2000
    x, w, A, B = rn(M, K), rn(N, K), rn(L, r, K), rn(L, N, r)
    scale, ids = torch.ones(L, device='cuda'), torch.randint(0, L, (M,), generator=g, device='cuda').to(torch.int32)

    def extra(f):
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = f()
        torch.cuda.synchronize()
        return out, torch.cuda.max_memory_allocated() - base
    size = lambda *ts: sum(t.numel() * t.element_size() for t in ts if t is not None)
    (y, t), held = extra(lambda: adapters.adapted_linear_forward(x, w, None, A, B, scale, ids))
    assert held - size(y, t) < 2 << 20                                       # a copy of x: 8 MB, of A: 131 MB
    dy = torch.randn_like(y)
    for need_dx in (True, False):
        out, held = extra(lambda: adapters.adapted_linear_backward(dy, x, t, w, A, B, scale, ids, need_dx=need_dx))
        assert held - size(*out) < size(B) + size(w) + (8 << 20)             # partial sums of every adapter: 396 MB


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', [1, 2, 4])
def test_few_rows_of_a_wider_view(M, dtype):
    """2,048 -> 1,024 at rank 16: rows of an odd pitch and an odd start, and an A that starts between four elements."""
    K, N, r, L = 2048, 1024, 16, 3
    g = torch.Generator().manual_seed(M)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    x, w, B = rn(M, K + 3)[:, 1:K + 1], rn(N, K) / K ** 0.5, rn(L, N, r)
    A = (rn(L * r * K + 1) / K ** 0.5)[1:].view(L, r, K)
    scale, ids = (0.5 + torch.rand(L, generator=g)).cuda(), torch.tensor([2, 0, -1, 1], dtype=torch.int32, device='cuda')[:M].contiguous()
    for a in (A, A.clone()):
        for v in (x, x.contiguous()):
            y, t = adapters.adapted_linear_forward(v, w, None, a, B, scale, ids)
            ry, rt, ey, et = oad.forward(_d(x), _d(w), None, _d(A), _d(B), _d(scale), ids.cpu().numpy())
            _near(y, ry, ey)
            _near(t, rt, et)
