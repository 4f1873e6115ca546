"""Workspace sizes of the low-rank adapters (no GPU): what a call with given operands needs, against the buffers that its form uses."""
import pytest

A16 = 1 << 20                                                        # an aligned address (only looked at)


def _al(v):
    return (v + 255) // 256 * 256


@pytest.mark.parametrize('bf16', [0, 1])
def test_forward_holds_copies_only_of_operands_that_are_copied(lib, bf16):
    z = 2 if bf16 else 4
    M, K, N, r, L = 4096, 2048, 1024, 64, 4096
    size = lambda x=A16, ldx=K, w=A16, a=A16, K=K: lib.hmf_adapted_linear_workspace_bytes_for(x, ldx, w, a, M, K, N, r, L, bf16)
    own = _al(M * r * 4) + 2 * _al(M * 4) + _al((L + 2) * 4)         # t, the rows' order and their adapters
    copies = {'x': _al(M * K * z), 'w': _al(N * K * z), 'a': _al(L * r * K * z)}
    assert size() == own and size(ldx=K + 16 // z) == own
    assert size(x=A16 + z) == size(ldx=K + 1) == own + copies['x']
    assert size(w=A16 + z) == own + copies['w'] and size(a=A16 + z) == own + copies['a']
    assert lib.hmf_adapted_linear_workspace_bytes(M, K, N, r, L, bf16) == own + sum(copies.values())      # enough for any operands
    Kp = (K - 1 + 128 // z - 1) // (128 // z) * (128 // z)
    assert Kp == K and size(K=K - 1) == own + sum(copies.values())   # an odd width is copied into whole chunks
    assert lib.hmf_adapted_linear_workspace_bytes_for(A16, K, A16, A16, 0, K, N, r, L, bf16) == 0


@pytest.mark.parametrize('bf16', [0, 1])
def test_backward_holds_partial_sums_of_adapters_with_many_rows_only(lib, bf16):
    z = 2 if bf16 else 4
    size = lambda M, L, dx, K=2048, N=1024, r=16: lib.hmf_adapted_linear_backward_workspace_bytes_for(M, K, N, r, L, bf16, dx)
    fixed = lambda M, L, K=2048, N=1024, r=16: _al(M * r * 4) + 2 * _al(M * 4) + _al((L + 2) * 4) + _al(L * r * N * z)      # u, order, adapters, B^T
    part = lambda p, K=2048, N=1024, r=16: _al(p * r * K * 4) + _al(p * r * N * 4)
    for M, L in ((4096, 1), (4096, 16), (4096, 4000), (257, 300), (300, 1)):
        most = 0                                                     # pieces of 256 rows of adapters that have more: all rows to as many of them as there can be
        for n in range(1, min(L, M // 257) + 1):
            rows = [M // n + (k < M % n) for k in range(n)]
            most = max(most, sum((v + 255) // 256 for v in rows if v > 256))
        p = min(L, M // 257) + M // 256
        assert most <= p and size(M, L, 0) == fixed(M, L) + part(p)
    assert size(4096, 16, 1) > size(4096, 16, 0) and size(200, 16, 1) > size(200, 16, 0)
    for M, L in ((4096, 16), (200, 16)):
        assert lib.hmf_adapted_linear_backward_workspace_bytes(M, 2048, 1024, 16, L, bf16) == size(M, L, 1)


@pytest.mark.parametrize('bf16', [0, 1])
def test_one_launch_goes_by_how_the_operands_lie(lib, bf16):
    """Four rows and 256 or 512 KB of A are one launch (no workspace) only where four elements are read at a time; up to 64 KB always."""
    z = 2 if bf16 else 4
    size = lambda x=A16, ldx=2048, w=A16, a=A16, K=2048, r=16, M=4: lib.hmf_adapted_linear_workspace_bytes_for(x, ldx, w, a, M, K, 1024, r, 3, bf16)
    assert size() == 0 and size(ldx=2052) == 0 and size(x=A16 + 4 * z) == 0
    assert size(ldx=2049) > 0 and size(x=A16 + z) > 0 and size(w=A16 + z) > 0 and size(a=A16 + z) > 0 and size(K=2047) > 0
    assert size(ldx=2049, r=1) == 0 and size(K=2047, ldx=2047, r=1) == 0 and size(M=5) > 0
    assert lib.hmf_adapted_linear_workspace_bytes(4, 2048, 1024, 16, 3, bf16) == size(ldx=2049)      # enough for any operands
