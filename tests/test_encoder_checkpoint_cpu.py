"""The encoder's choice of checkpoint is checked before anything runs (no GPU)."""
import pytest
import torch

from humaniflow_amd.encoder import ResNetEncoder
from humaniflow_amd.encoder_train import EncoderTrainFn


@pytest.mark.parametrize('mode', ['fp8', 'INT8', 8, True])
def test_an_unknown_checkpoint_is_refused(mode):
    enc = ResNetEncoder(18, 18).train()
    enc.activation_checkpoint = mode
    with pytest.raises(ValueError, match='activation_checkpoint'):
        EncoderTrainFn.apply(enc, torch.zeros(1, 18, 64, 64), *enc.parameters())
