"""Models whose forward knows nothing of adapters (a wrapper, a subclass with its own forward) go through the drivers as before: without ids none are passed (no GPU)."""
import pytest
import torch

from humaniflow_amd import evaluate, predict, train


class Reached(Exception):
    pass


class Plain:
    """Takes what the drivers passed before there were adapters."""
    pose_so3flow_transform_modules = torch.nn.ModuleList()

    def eval(self):
        return self

    def __call__(self, input, compute_point_est=True, num_samples=0, use_shape_mode_for_samples=False, compute_for_loglik=False, shape_for_loglik=None,
                 pose_R_for_loglik=None, glob_R_for_loglik=None, input_feats=None, return_input_feats=False, noise=None):
        raise Reached


class Adapted(Plain):
    def __call__(self, input, adapter_ids, **kw):
        raise Reached(adapter_ids.tolist())


CALLS = {'predict': lambda m, **kw: predict.predict_humaniflow(m, None, torch.zeros(2, 18, 8, 8), ['a', 'b'], **kw),
         'evaluate': lambda m, **kw: evaluate.predict_batch(m, None, {'input': torch.zeros(2, 18, 8, 8)}, 0, **kw),
         'train': lambda m, **kw: train.train_forward_loss(m, None, None, torch.zeros(2, 18, 8, 8), dict(shape=None, pose_rotmats=None, glob_rotmats=None), 1, **kw)}


@pytest.mark.parametrize('name', sorted(CALLS))
def test_no_ids_are_passed_where_none_are_given(name):
    with pytest.raises(Reached):
        CALLS[name](Plain())
    with pytest.raises(Reached, match=r'\[3\]' if name == 'predict' else '3, -1'):
        CALLS[name](Adapted(), adapter_ids=torch.tensor([3, -1]))
