"""What a pass through adapted layers keeps when their inputs are kept in 8 bits."""
import pytest
import torch

import humaniflow_amd as H
from humaniflow_amd import act8, adapters
from helpers import init_model_for_tests

pytestmark = pytest.mark.gpu


def _args(M=400, K=512, N=48, r=4, L=3):
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g).cuda()
    return rn(M, K), (rn(N, K) / K ** 0.5, rn(N), rn(L, r, K).requires_grad_(True), rn(L, N, r).requires_grad_(True), torch.ones(L, device='cuda'),
                      torch.randint(-1, L, (M,), generator=g).to(torch.int32).cuda())


def test_a_checkpoint_made_before_is_shared():
    """Two layers on one x: the gradients with one shared checkpoint are those with one each, bit for bit."""
    x, (w, b, A, B, scale, ids) = _args()
    got = []
    for ck in ('int8', act8.pack(x)):
        y = sum(adapted.sum() * k for k, adapted in enumerate(adapters.adapted_linear(x, w, b, A, B, scale, ids, checkpoint=ck) for _ in range(2)))
        got.append(torch.autograd.grad(y, (A, B)))
    assert all(torch.equal(p, q) for p, q in zip(*got))
    with pytest.raises(ValueError, match='checkpoint holds'):
        adapters.adapted_linear(x, w, b, A, B, scale, ids, checkpoint=act8.pack(x[:32]))
    with pytest.raises(ValueError, match='checkpoint must be'):
        adapters.adapted_linear(x, w, b, A, B, scale, ids, checkpoint='int4')


def test_the_models_heads_keep_one_checkpoint_of_their_common_input(monkeypatch):
    cfg = H.get_humaniflow_cfg_defaults()
    model = init_model_for_tests(H.HumaniflowModel(torch.device('cpu'), cfg.MODEL, H.SMPL_PARENTS), seed=1).cuda().eval().requires_grad_(False)
    feats, ids = torch.randn(9, 512, device='cuda'), torch.arange(9, device='cuda').to(torch.int32) % 3 - 1
    made = []
    real = act8.pack
    monkeypatch.setattr(act8, 'pack', lambda x: made.append(tuple(x.shape)) or real(x))

    def packs(checkpoint, layers=H.LowRankAdapters.HEADS, grad=True):
        torch.manual_seed(0)
        model.attach_adapters(H.LowRankAdapters(model, 2, 4, checkpoint=checkpoint, layers=layers))
        made.clear()
        with torch.set_grad_enabled(grad):
            out = model(None, input_feats=feats, adapter_ids=ids, compute_point_est=False)
        model.attach_adapters(None)
        assert out['cam_wp'].requires_grad == grad
        return len(made)
    assert packs('int8') == 2                                        # fc1's input and the three heads'
    assert packs('int8', layers=('fc1',)) == 1 and packs('int8', layers=('fc_cam', 'fc_shape')) == 1
    assert packs('int8', grad=False) == 0 and packs(None) == 0


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
