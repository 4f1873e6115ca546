"""Low-rank adapters without a GPU: the oracle's gradients against differences, and what the entry points refuse."""
import ctypes as C

import numpy as np
import pytest
import torch

import humaniflow_amd as H
from humaniflow_amd import adapters
from oracle import adapters as oad


def test_oracle_gradients_against_differences():
    """y is linear in each of x, A and B: central differences are exact up to rounding (1e-16 / 1e-3 of values of order 1)."""
    rng = np.random.default_rng(0)
    M, K, N, r, L = 6, 5, 4, 2, 3
    x, w, bias, a, b = (rng.standard_normal(s) for s in ((M, K), (N, K), (N,), (L, r, K), (L, N, r)))
    scale, ids, dy = rng.uniform(0.5, 2, L), np.array([2, -1, 0, 2, 2, -7]), rng.standard_normal((M, N))
    f = lambda x, a, b: (dy * oad.forward(x, w, bias, a, b, scale, ids)[0]).sum()
    _, t, _, _ = oad.forward(x, w, bias, a, b, scale, ids)
    dx, da, db, *_ = oad.backward(dy, x, t, w, a, b, scale, ids)
    assert not da[1].any() and not db[1].any()
    h = 1e-3
    for k, (v, g) in enumerate(((x, dx), (a, da), (b, db))):
        for at in np.ndindex(v.shape):
            d = np.zeros_like(v)
            d[at] = h
            args = [x, a, b]
            hi, lo = list(args), list(args)
            hi[k], lo[k] = v + d, v - d
            assert abs((f(*hi) - f(*lo)) / (2 * h) - g[at]) < 1e-9


def _args(M=4, K=6, N=3, r=2, L=2, dt=torch.float32):
    f = torch.zeros
    return dict(x=f(M, K, dtype=dt), weight=f(N, K, dtype=dt), bias=f(N, dtype=dt), A=f(L, r, K, dtype=dt), B=f(L, N, r, dtype=dt), scale=f(L), ids=f(M, dtype=torch.int32))


def test_refusals_of_the_python_entry_points():
    f = torch.zeros
    for change, match in ((dict(x=f(4, 5)), 'do not fit'), (dict(A=f(2, 2, 5)), 'do not fit'), (dict(B=f(2, 3, 3)), 'do not fit'), (dict(bias=f(4)), 'bias'),
                          (dict(A=f(2, 65, 6), B=f(2, 3, 65)), 'rank 65'), (dict(scale=f(3)), 'scale'), (dict(scale=f(2).double()), 'scale'), (dict(ids=f(4)), 'ids'),
                          (dict(ids=f(3, dtype=torch.int32)), 'ids'), (dict(weight=f(3, 6).half()), 'float32 and bfloat16'), (dict(A=f(2, 2, 6).bfloat16()), 'type'),
                          (dict(x=f(4, 6, 1)), 'takes x'), (dict(A=f(0, 2, 6), B=f(0, 3, 2), scale=f(0)), 'do not fit')):
        with pytest.raises(ValueError, match=match):
            adapters.adapted_linear(**{**_args(), **change})
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        adapters.adapted_linear(**_args())
    with pytest.raises(ValueError, match='checkpoint'):
        adapters.adapted_linear(**_args(), checkpoint='int4')
    a = _args()
    a['weight'].requires_grad_(True)
    with pytest.raises(RuntimeError, match='fixed projection'):
        adapters.adapted_linear(**a)


def test_refusals_of_the_c_entry_points(lib):
    buf = (C.c_float * 4096)()
    p = C.c_void_p((C.addressof(buf) + 15) & ~15)
    n = C.c_void_p(None)
    need = lib.hmf_adapted_linear_workspace_bytes(5, 6, 3, 2, 2, 0)
    assert lib.hmf_adapted_linear_workspace_bytes(4, 6, 3, 2, 2, 0) == 0      # one launch
    fw = lambda x=p, ldx=6, M=5, K=6, N=3, r=2, L=2, ws=p, nb=1 << 20: lib.hmf_adapted_linear(x, ldx, p, n, p, p, p, p, M, K, N, r, L, 0, p, n, ws, nb, n)
    assert need > 0 and fw(M=0) == 0
    assert fw(x=n) == -1 and fw(ldx=5) == -1 and fw(K=0) == -1 and fw(M=-1) == -1 and fw(L=0) == -1 and fw(r=0) == -1
    assert fw(r=65) == -2 and fw(L=70000) == -2
    assert fw(M=256, N=1 << 25) == -2 and fw(M=1 << 25) == -2 and b'grid' in lib.hmf_last_error()
    assert fw(ws=n) == -4 and fw(nb=need - 1) == -4 and fw(ws=C.c_void_p(p.value + 4)) == -4
    need = lib.hmf_adapted_linear_backward_workspace_bytes(4, 6, 3, 2, 2, 0)
    bw = lambda dy=p, ldx=6, exps=n, M=4, r=2, ws=p, nb=1 << 20: lib.hmf_adapted_linear_backward(dy, p, ldx, exps, p, p, p, p, p, p, M, 6, 3, r, 2, 0, p, p, p, ws, nb, n)
    assert bw(dy=n) == -1 and bw(ldx=5) == -1 and bw(ldx=7, exps=p) == -1 and bw(M=0) == -1 and bw(r=65) == -2 and bw(nb=need - 1) == -4 and bw(ws=n) == -4
    assert lib.hmf_adapted_linear_workspace_bytes(0, 6, 3, 2, 2, 0) == 0
    assert fw(L=65535, N=1 << 17) == -2 and b'grid' in lib.hmf_last_error()      # a work-group of the gradients per adapter and 128 columns


def test_module_layout_and_refusals():
    cfg = H.get_humaniflow_cfg_defaults()
    model = H.HumaniflowModel(torch.device('cpu'), cfg.MODEL, H.SMPL_PARENTS)
    plain = set(model.state_dict())
    ad = H.LowRankAdapters(model, 3, 4, alpha=8, layers=('fc1', 'fc_shape'))
    assert set(ad.state_dict()) == {'scale', 'fc1_A', 'fc1_B', 'fc_shape_A', 'fc_shape_B'}
    assert tuple(ad.fc1_A.shape) == (3, 4, 512) and tuple(ad.fc_shape_B.shape) == (3, 20, 4) and ad.scale.tolist() == [2.0] * 3 and not ad.fc1_B.any()
    model.attach_adapters(ad)
    assert set(model.state_dict()) == plain | {'adapters.' + k for k in ad.state_dict()}
    model.attach_adapters(None)
    assert set(model.state_dict()) == plain                                # the reference's checkpoint layout again
    for bad in (dict(num_adapters=0, rank=4), dict(num_adapters=1, rank=0), dict(num_adapters=1, rank=65), dict(num_adapters=1, rank=1, layers=('conv1',)),
                dict(num_adapters=1, rank=1, layers=()), dict(num_adapters=1, rank=1, checkpoint='fp8')):
        with pytest.raises(ValueError):
            H.LowRankAdapters(model, **bad)
    with pytest.raises(RuntimeError, match='no adapters'):
        model(torch.zeros(1, 18, 64, 64), adapter_ids=torch.zeros(1, dtype=torch.int32))
    wrong = H.get_benchmark_cfg()
    with pytest.raises(ValueError, match='do not fit'):
        H.HumaniflowModel(torch.device('cpu'), wrong.MODEL, H.SMPL_PARENTS).attach_adapters(ad)
