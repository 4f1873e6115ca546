"""Capturing the encoder's training pass beside a living eager pass over the same parameters: the check itself, without a capture."""
import pytest
import torch

from humaniflow_amd.encoder import ResNetEncoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('checkpoint', [None, 'int8'])
def test_capture_beside_a_living_eager_pass_is_refused(monkeypatch, checkpoint):
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.activation_checkpoint = checkpoint
    x = torch.randn(2, 18, 64, 64, device='cuda')
    f = enc(x)                                                       # alive, on the default stream
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        with pytest.raises(RuntimeError, match='still alive'):
            enc(x)
    f.sum().backward()
    del f
    with monkeypatch.context() as m:                                 # let go of: allowed
        m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        enc(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f = enc(x)                                                   # alive on a stream that a capture can wait for
    torch.cuda.current_stream().wait_stream(side)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        enc(x)


def test_a_frozen_first_layer_is_no_obstacle(monkeypatch):
    torch.manual_seed(0)
    enc = ResNetEncoder(18, 18).cuda().train()
    enc.conv1.requires_grad_(False)
    x = torch.randn(2, 18, 64, 64, device='cuda')
    f = enc(x)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='still alive'):
        enc(x)
    del f
    enc(x)
