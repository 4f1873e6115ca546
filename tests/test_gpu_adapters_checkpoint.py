"""What a pass through adapted layers keeps when their inputs are kept in 8 bits."""
import pytest
import torch

from humaniflow_amd import adapters

pytestmark = pytest.mark.gpu


def _args(M=400, K=512, N=48, r=4, L=3):
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g).cuda()
    return rn(M, K), (rn(N, K) / K ** 0.5, rn(N), rn(L, r, K).requires_grad_(True), rn(L, N, r).requires_grad_(True), torch.ones(L, device='cuda'),
                      torch.randint(-1, L, (M,), generator=g).to(torch.int32).cuda())


def test_the_checkpoint_is_let_go_of_by_the_backward_pass():
    """Like every saved tensor: with the output still alive, and a second backward pass is refused."""
    x, (w, b, A, B, scale, ids) = _args(M=40000)
    y = adapters.adapted_linear(x, w, b, A, B, scale, ids, checkpoint='int8')
    loss = y.sum()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    loss.backward()
    grads = A.grad.numel() * 4 + B.grad.numel() * 4
    assert held + grads - torch.cuda.memory_allocated() > x.numel()      # a byte per element and more
    with pytest.raises(RuntimeError, match='second time'):
        loss.backward()
