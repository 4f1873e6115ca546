"""Capturing the encoder's training pass beside a living eager pass over the same parameters: the check itself, without a capture."""
import pytest
import torch

from humaniflow_amd.encoder import ResNetEncoder

pytestmark = pytest.mark.gpu


def _captured_backward(enc, x, monkeypatch):
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        f = enc(x)                                                   # a forward pass alone is no obstacle
        return torch.autograd.grad(f.sum(), [p for p in enc.parameters() if p.requires_grad])


@pytest.mark.parametrize('checkpoint', [None, 'int8'])
def test_capture_beside_a_living_eager_pass_is_refused(monkeypatch, checkpoint):
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.activation_checkpoint = checkpoint
    x = torch.randn(2, 18, 64, 64, device='cuda')
    f = enc(x)                                                       # alive, on the default stream
    with pytest.raises(RuntimeError, match='still alive'):
        _captured_backward(enc, x, monkeypatch)
    f.sum().backward()
    del f
    assert len(_captured_backward(enc, x, monkeypatch)) > 50         # let go of: allowed
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f = enc(x)                                                   # alive on a stream that a capture can wait for
    torch.cuda.current_stream().wait_stream(side)
    assert len(_captured_backward(enc, x, monkeypatch)) > 50


def test_a_frozen_first_layer_is_no_obstacle(monkeypatch):
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.conv1.requires_grad_(False)
    x = torch.randn(2, 18, 64, 64, device='cuda')
    f = enc(x)
    with pytest.raises(RuntimeError, match='still alive'):
        _captured_backward(enc, x, monkeypatch)
    del f
    assert len(_captured_backward(enc, x, monkeypatch)) > 50


def test_parameters_that_are_not_leaves():
    """Substituted parameters that were computed from others: there is nothing to note, and the forward pass runs."""
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    x = torch.randn(2, 18, 64, 64, device='cuda')
    base = {n: p.detach().clone().requires_grad_(True) for n, p in enc.named_parameters()}
    f = torch.func.functional_call(enc, {n: p * 1.0 for n, p in base.items()}, (x,))
    assert f.requires_grad and torch.isfinite(f).all()
