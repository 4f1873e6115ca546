"""8-bit activation checkpoints without a GPU: the oracle's definition against its own bounds and against finite differences, and what the entry points refuse."""
import ctypes as C

import numpy as np
import pytest
import torch

from humaniflow_amd import act8
from oracle import act8 as oact


@pytest.mark.parametrize('seed', range(4))
def test_oracle_rounding_is_at_most_half_a_step(seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((70, 9)) * np.exp2(rng.integers(-30, 30, 9))).astype(np.float32).astype(np.float64)
    codes, exps = oact.pack(x)
    v = oact.values(codes, exps)
    step = np.exp2(exps.astype(np.float64)).repeat(32, axis=0)[:70]
    assert np.all(np.abs(v - x) <= step / 2)
    top = np.stack([np.abs(x[t * 32:(t + 1) * 32]).max(axis=0) for t in range(3)])
    assert np.all(top / np.exp2(exps) < 127.5) and np.all(top / np.exp2(exps) >= 63.5)


def test_oracle_bn_backward_is_the_gradient():
    """Against central differences of sum(g * relu(gamma xhat(y) + beta + idt)) in float64 (step 1e-6: truncation 1e-12, rounding 1e-10)."""
    rng = np.random.default_rng(0)
    M, Cn = 12, 3
    y, idt, g = rng.standard_normal((M, Cn)), rng.standard_normal((M, Cn)), rng.standard_normal((M, Cn))
    gamma, beta, eps = rng.uniform(0.5, 1.5, Cn), rng.standard_normal(Cn), 1e-5

    def f(y, gamma, beta):
        mean, var = y.mean(axis=0), y.var(axis=0)
        return (g * np.maximum(gamma * (y - mean) / np.sqrt(var + eps) + beta + idt, 0)).sum()
    mean, rstd = y.mean(axis=0), 1 / np.sqrt(y.var(axis=0) + eps)
    xhat = (y - mean) * rstd
    _, gg, gb, gy = oact.bn_backward(g, xhat, gamma * xhat + beta + idt > 0, rstd, gamma)
    h = 1e-6
    for m in range(M):
        for c in range(Cn):
            d = np.zeros_like(y)
            d[m, c] = h
            assert abs((f(y + d, gamma, beta) - f(y - d, gamma, beta)) / (2 * h) - gy[m, c]) < 1e-7
    for c in range(Cn):
        d = np.zeros(Cn)
        d[c] = h
        assert abs((f(y, gamma + d, beta) - f(y, gamma - d, beta)) / (2 * h) - gg[c]) < 1e-7
        assert abs((f(y, gamma, beta + d) - f(y, gamma, beta - d)) / (2 * h) - gb[c]) < 1e-7


def test_refusals_of_the_python_entry_points():
    f = torch.zeros
    ck = act8.Act8(f(40, 64, dtype=torch.int8), f(2, 64, dtype=torch.uint8))
    assert ck.nbytes() == 40 * 64 + 2 * 64 and tuple(ck.shape) == (40, 64)
    with pytest.raises(ValueError, match='exps'):
        act8.Act8(f(40, 64, dtype=torch.int8), f(1, 64, dtype=torch.uint8))
    with pytest.raises(ValueError, match='Act8 takes'):
        act8.Act8(f(40, 64), f(2, 64, dtype=torch.uint8))
    with pytest.raises(ValueError, match='contiguous'):
        act8.Act8(f(64, 40, dtype=torch.int8).t(), f(2, 64, dtype=torch.uint8))
    for call in (lambda: act8.pack(f(4, 4)), lambda: act8.unpack(ck), lambda: act8.bn_apply(f(4, 64), f(64), f(64)),
                 lambda: act8.restore_activation(ck, f(64), f(64)), lambda: act8.bn_backward(f(40, 64), ck, None, f(64), f(64), f(64))):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()
    with pytest.raises(ValueError, match='float32 or bfloat16'):
        act8.unpack(ck, dtype=torch.float16)
    with pytest.raises(ValueError, match='float32'):
        act8.bn_apply(f(4, 64, dtype=torch.bfloat16), f(64), f(64))


def test_refusals_of_the_c_entry_points(lib):
    """Arguments are checked before any launch: no GPU needed."""
    buf = (C.c_float * 4096)()
    p = C.c_void_p((C.addressof(buf) + 15) & ~15)
    odd = C.c_void_p(p.value + 4)
    n = C.c_void_p(None)
    assert lib.hmf_act8_pack(p, 3, 0, 2, 4, p, p, n) == -1 and b'ld=3' in lib.hmf_last_error()
    assert lib.hmf_act8_pack(n, 4, 0, 2, 4, p, p, n) == -1
    assert lib.hmf_act8_pack(p, 4, 0, -1, 4, p, p, n) == -1
    assert lib.hmf_act8_pack(n, 4, 0, 0, 4, n, n, n) == 0                       # no rows: nothing to do
    assert lib.hmf_act8_unpack(p, p, 2, -3, p, 0, n) == -1
    assert lib.hmf_act8_unpack(p, n, 2, 3, p, 0, n) == -1
    assert lib.hmf_act8_pack(p, 4, 0, 0x7fffffff, 4, p, p, n) == -2 and lib.hmf_act8_unpack(p, p, 0x7fffff00, 0x7fffff00, p, 0, n) == -2
    bn = lambda y=p, bits=p, oc=n, oe=n, M=2, Cn=64, relu=1: lib.hmf_bn_apply_act8(y, p, p, n, p, p, p, bits, oc, oe, M, Cn, relu, n)
    assert bn(Cn=63) == -1 and bn(M=0) == -1 and bn(y=n) == -1 and bn(bits=n) == -1 and bn(relu=0) == -1 and bn(oc=p) == -1 and bn(oe=p) == -1
    assert bn(y=odd) == -1 and b'aligned' in lib.hmf_last_error()
    assert lib.hmf_act8_restore_activation(p, p, n, p, p, p, 2, 65, n) == -1
    assert lib.hmf_act8_restore_activation(p, p, odd, p, p, p, 2, 64, n) == -1
    need = lib.hmf_bn_backward_act8_workspace_bytes(100, 64)
    assert need > 0 and lib.hmf_bn_backward_act8_workspace_bytes(100, 60) == 0
    bw = lambda g=p, Cn=64, ws=p, nb=need: lib.hmf_bn_backward_act8(g, p, p, n, p, p, p, p, n, p, p, 100, Cn, ws, nb, n)
    assert bw(Cn=32) == -1 and bw(g=odd) == -1 and bw(ws=n) == -4 and bw(nb=need - 1) == -4


def test_encoder_refuses_an_unknown_checkpoint():
    from humaniflow_amd.encoder import ResNetEncoder
    assert ResNetEncoder.activation_checkpoint is None
