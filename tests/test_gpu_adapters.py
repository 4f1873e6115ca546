"""Low-rank adapters on the device against their definition in 64 bits (oracle/adapters.py, which also derives what 32-bit sums may be off by); a bfloat16 result is
rounded once more, by at most 2^-8 of its value (half a step is 2^-9; the other half covers a value whose 32-bit error moved it over a rounding border)."""
import numpy as np
import pytest
import torch

import humaniflow_amd as H
from humaniflow_amd import act8, adapters
from helpers import init_model_for_tests
from oracle import act8 as oact
from oracle import adapters as oad

pytestmark = pytest.mark.gpu


def _case(M, K, N, r, L, kind, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    c = dict(x=rn(M, K), weight=rn(N, K) / K ** 0.5, bias=rn(N), A=rn(L, r, K) / K ** 0.5, B=rn(L, N, r) / r ** 0.5)
    c = {k: v.to(dtype).cuda() for k, v in c.items()}
    c['scale'] = (0.5 + torch.rand(L, generator=g)).cuda()
    if kind == 'one':
        ids = torch.full((M,), L - 1)
    elif kind == 'none':
        ids = torch.full((M,), -1)
    elif kind == 'runs':
        ids = (torch.arange(M) * (L + 1) // max(M, 1)) - 1
    else:
        ids = torch.randint(-1, L, (M,), generator=g)
    c['ids'] = ids.to(torch.int32).cuda()
    return c


def _d(t):
    return t.double().cpu().numpy()


def _near(got, ref, bound):
    got = got.detach()
    tol = bound + (2.0 ** -8 * np.abs(ref) if got.dtype == torch.bfloat16 else 0.0) + 1e-37
    got = _d(got)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = np.isnan(ref) | (np.abs(got - ref) <= tol)
    assert ok.all(), (np.abs(got - ref)[~ok].max(), np.argwhere(~ok)[:4].tolist(), (~ok).sum())


def _check_forward(c):
    y, t = adapters.adapted_linear_forward(**c)
    ry, rt, ey, et = oad.forward(_d(c['x']), _d(c['weight']), None if c['bias'] is None else _d(c['bias']), _d(c['A']), _d(c['B']), _d(c['scale']), c['ids'].cpu().numpy())
    _near(y, ry, ey)
    _near(t, rt, et)
    return y, t


def _check_backward(c, x8=False, seed=0):
    M, N = c['x'].shape[0], c['weight'].shape[0]
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(seed + 77)).to(c['x'].dtype).cuda()
    ck = act8.pack(c['x']) if x8 else None
    x = _d(act8.unpack(ck)) if x8 else _d(c['x'])
    t = adapters.adapted_linear_forward(**c)[1]
    dx, dA, dB = adapters.adapted_linear_backward(dy, ck if x8 else c['x'], t, c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    rx, ra, rb, ex, ea, eb = oad.backward(_d(dy), x, _d(t), _d(c['weight']), _d(c['A']), _d(c['B']), _d(c['scale']), c['ids'].cpu().numpy())
    _near(dx, rx, ex)
    _near(dA, ra, ea)
    _near(dB, rb, eb)
    none, dA2, dB2 = adapters.adapted_linear_backward(dy, ck if x8 else c['x'], t, c['weight'], c['A'], c['B'], c['scale'], c['ids'], need_dx=False)
    assert none is None and torch.equal(dA, dA2) and torch.equal(dB, dB2)
    return dx, dA, dB


SHAPES = [(1, 32, 3, 1, 1, 'one'), (1, 2048, 1024, 16, 1, 'one'), (2, 33, 5, 3, 4, 'mixed'), (32, 1024, 20, 4, 32, 'mixed'), (33, 64, 65, 64, 2, 'runs'),
          (72, 512, 512, 8, 12, 'mixed'), (255, 100, 70, 5, 9, 'mixed'), (256, 128, 128, 33, 3, 'runs'), (40, 96, 32, 16, 5, 'none'),
          (257, 128, 128, 16, 3, 'mixed'), (300, 72, 130, 7, 50, 'mixed'), (1000, 256, 384, 16, 8, 'runs'), (513, 515, 77, 12, 5, 'mixed'), (700, 64, 192, 64, 1, 'one'),
          (640, 192, 64, 4, 70, 'mixed'), (400, 160, 96, 8, 4, 'none'), (1111, 2048, 264, 9, 200, 'mixed')]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,r,L,kind', SHAPES)
def test_forward(M, K, N, r, L, kind, dtype):
    _check_forward(_case(M, K, N, r, L, kind, dtype, M + K + N))


@pytest.mark.parametrize('x8', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K,N,r,L,kind', SHAPES)
def test_backward(M, K, N, r, L, kind, dtype, x8):
    _check_backward(_case(M, K, N, r, L, kind, dtype, M + K + N), x8)


@pytest.mark.parametrize('M', [3, 70, 400])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strides_alignment_and_no_bias(M, dtype):
    """Rows of wider rows, unaligned starts, transposed and expanded inputs, 64-bit ids: the results of the contiguous copies."""
    K, N = 96, 64
    c = _case(M, K, N, 8, 3, 'mixed', dtype, M)
    c['bias'] = None
    ref, reft = _check_forward(c)
    wide = torch.empty(M, K + 9, dtype=dtype, device='cuda')
    for off in (0, 1, 8):
        wide[:, off:off + K] = c['x']
        y, t = adapters.adapted_linear_forward(**{**c, 'x': wide[:, off:off + K]})
        ry, rt, ey, et = oad.forward(_d(c['x']), _d(c['weight']), None, _d(c['A']), _d(c['B']), _d(c['scale']), c['ids'].cpu().numpy())
        _near(y, ry, ey)
        _near(t, rt, et)
    y = adapters.adapted_linear(**{**c, 'x': c['x'].t().contiguous().t(), 'weight': c['weight'].t().contiguous().t(), 'ids': c['ids'].long()})
    assert torch.equal(y, ref)
    one = adapters.adapted_linear(**{**c, 'x': c['x'][:1].expand(M, K)})
    _near(one, *[v for v in oad.forward(_d(c['x'][:1]).repeat(M, 0), _d(c['weight']), None, _d(c['A']), _d(c['B']), _d(c['scale']), c['ids'].cpu().numpy())][::2])


@pytest.mark.parametrize('M', [5, 300])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_one_requests_infinities_stay_its_own(M, dtype):
    """An adapter with infinite or NaN weights, rows with NaN, ids that no adapter has: nothing of them reaches other rows or other adapters' gradients."""
    c = _case(M, 64, 48, 4, 4, 'mixed', dtype, 3)
    c['ids'] = (torch.arange(M) % 5 - 1).to(torch.int32).cuda()
    clean, _ = adapters.adapted_linear_forward(**c)
    t = adapters.adapted_linear_forward(**c)[1]
    dy = torch.randn(M, 48, device='cuda').to(dtype)
    args = lambda: (c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    cdx, cdA, cdB = adapters.adapted_linear_backward(dy, c['x'], t, *args())
    c['B'][2, 7, 1], c['B'][2, 9, 0], c['A'][2, 0, 5] = float('nan'), float('inf'), float('-inf')
    y, tt = adapters.adapted_linear_forward(**c)
    other = (c['ids'] != 2).cpu()
    assert torch.equal(y[other], clean[other])
    rows = ~other
    assert not torch.isfinite(y[rows][:, 7]).any() and not torch.isfinite(y[rows][:, 9]).any()
    dx, dA, dB = adapters.adapted_linear_backward(dy, c['x'], t, *args())
    assert torch.equal(dx[other], cdx[other]) and all(torch.equal(dA[l], cdA[l]) and torch.equal(dB[l], cdB[l]) for l in (0, 1, 3))
    c = _case(M, 64, 48, 4, 4, 'mixed', dtype, 3)
    c['ids'][1], c['ids'][3] = 4, 2 ** 31 - 1
    c['x'][2, 0] = float('nan')
    y, t = _check_forward(c)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isnan(y[2]).all()
    c['x'][2, 0] = 0.0
    _check_backward(c)


def test_infinite_weight_of_one_rank_is_added_to_its_rows():
    """inf times a positive t is inf, not NaN, in both forms."""
    for M in (6, 300):
        c = _case(M, 64, 48, 4, 2, 'one', torch.bfloat16, 1)
        c['ids'] = (torch.arange(M) % 2).to(torch.int32).cuda()
        c['B'][1, 5, 2] = float('inf')
        y, t = adapters.adapted_linear_forward(**c)
        rows = (c['ids'] == 1)
        want = torch.where(t[rows][:, 2] > 0, float('inf'), float('-inf'))
        assert torch.equal(y[rows][:, 5].float(), want) and torch.isfinite(y[~rows]).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', [6, 300])
def test_infinite_gradient_of_one_output(M, dtype):
    """An infinity in dy is one in the gradients that it reaches (times t, u and x that are not zero), in both forms, and reaches no other adapter."""
    c = _case(M, 64, 48, 4, 2, 'one', dtype, 1)
    c['ids'] = (torch.arange(M) % 2).to(torch.int32).cuda()
    t = adapters.adapted_linear_forward(**c)[1]
    dy = torch.randn(M, 48, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    args = (c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    _, cA, cB = adapters.adapted_linear_backward(dy, c['x'], t, *args)
    dy[1, 5] = float('inf')
    _, dA, dB = adapters.adapted_linear_backward(dy, c['x'], t, *args)
    assert torch.equal(dA[0], cA[0]) and torch.equal(dB[0], cB[0])
    inf = torch.full((), float('inf'), device='cuda', dtype=dtype)
    assert torch.equal(dB[1, 5], torch.copysign(inf, t[1].to(dtype))) and torch.equal(dB[1, 6:], cB[1, 6:]) and torch.equal(dB[1, :5], cB[1, :5])
    assert torch.equal(dA[1], torch.copysign(inf, c['B'][1, 5][:, None] * c['x'][1][None, :]))


def test_empty_and_refused():
    c = _case(4, 64, 48, 4, 2, 'mixed', torch.float32, 0)
    y = adapters.adapted_linear(**{**c, 'x': c['x'][:0], 'ids': c['ids'][:0]})
    assert tuple(y.shape) == (0, 48)
    dx, dA, dB = adapters.adapted_linear_backward(y, c['x'][:0], torch.empty(0, 4, device='cuda'), c['weight'], c['A'], c['B'], c['scale'], c['ids'][:0])
    assert tuple(dx.shape) == (0, 64) and not dA.any() and not dB.any()
    with pytest.raises(ValueError, match='is on cpu'):
        adapters.adapted_linear(**{**c, 'ids': c['ids'].cpu()})
    with pytest.raises(ValueError, match='x is'):
        adapters.adapted_linear(**{**c, 'x': c['x'].bfloat16()})
    t = torch.zeros(4, 4, device='cuda')
    with pytest.raises(ValueError, match='`t`'):
        adapters.adapted_linear_backward(torch.zeros(4, 48, device='cuda'), c['x'], t[:, :3], c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    with pytest.raises(ValueError, match='`dy`'):
        adapters.adapted_linear_backward(torch.zeros(4, 47, device='cuda'), c['x'], t, c['weight'], c['A'], c['B'], c['scale'], c['ids'])


@pytest.mark.parametrize('M', [20, 400])
@pytest.mark.parametrize('checkpoint', [None, 'int8'])
def test_autograd_gradients_and_differences(M, checkpoint):
    c = _case(M, 64, 40, 4, 3, 'mixed', torch.float32, 5)
    leaf = {k: c[k].clone().requires_grad_(True) for k in ('x', 'A', 'B')}
    w = torch.randn(M, 40, device='cuda')
    (adapters.adapted_linear(**{**c, **leaf}, checkpoint=checkpoint) * w).sum().backward()
    x = act8.unpack(act8.pack(c['x'])) if checkpoint else c['x']
    t = adapters.adapted_linear_forward(**c)[1]
    dx, dA, dB = adapters.adapted_linear_backward(w, x, t, c['weight'], c['A'], c['B'], c['scale'], c['ids'])
    assert torch.equal(leaf['x'].grad, dx) and torch.equal(leaf['A'].grad, dA) and torch.equal(leaf['B'].grad, dB)
    if checkpoint is None:                                               # y is linear in each: differences of the 64-bit definition along a random direction
        host = {k: _d(v) for k, v in c.items() if k != 'ids'}
        ids = c['ids'].cpu().numpy()
        f = lambda **k: (_d(w) * oad.forward(**{**{n: host[n] for n in ('x', 'scale')}, 'w': host['weight'], 'bias': host['bias'], 'a': host['A'], 'b': host['B'], 'ids': ids, **k})[0]).sum()
        for name, key in (('x', 'x'), ('A', 'a'), ('B', 'b')):
            d = np.random.default_rng(1).standard_normal(host[name].shape)
            diff = (f(**{key: host[name] + d}) - f(**{key: host[name] - d})) / 2
            g = _d(leaf[name].grad)
            # each of the n gradient entries is off by at most 1e-5 of the norm of its terms (see the oracle's bounds): the sum along d by sqrt(n) of that
            assert abs(diff - (g * d).sum()) <= 1e-5 * np.linalg.norm(g) * np.linalg.norm(d)


def test_streams_repeats_and_graph_replays():
    for M in (24, 500):
        c = _case(M, 256, 192, 8, 6, 'mixed', torch.bfloat16, 2)
        dy = torch.randn(M, 192, device='cuda').bfloat16()

        def step():
            y, t = adapters.adapted_linear_forward(**c)
            return [y, t, *adapters.adapted_linear_backward(dy, act8.pack(c['x']), t, c['weight'], c['A'], c['B'], c['scale'], c['ids'])]
        ref = [v.clone() for v in step()]
        assert all(torch.equal(a, b) for a, b in zip(ref, step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        here = step()                                                     # two at once
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) and torch.equal(a, d) for a, b, d in zip(ref, got, here))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for k in range(3):
            c['x'].mul_(0.9)
            c['ids'].copy_(torch.randint(-1, 6, (M,), device='cuda'))     # another mixture in the same graph
            want = [v.clone() for v in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, held)), (M, k)


@pytest.mark.parametrize('checkpoint', [None, 'int8'])
def test_captured_fit(checkpoint):
    """Forward and backward through autograd in one graph, replayed between the program's own passes; the kernels add in a fixed order, so the results are the same bits."""
    c = _case(300, 96, 64, 8, 3, 'mixed', torch.float32, 9)
    w = torch.randn(300, 64, device='cuda')
    leaf = {k: c[k].clone().requires_grad_(True) for k in ('x', 'A', 'B')}

    def step():
        y = adapters.adapted_linear(**{**c, **leaf}, checkpoint=checkpoint)
        return [y.detach(), *torch.autograd.grad((y * w).sum(), list(leaf.values()))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            leaf['x'].mul_(0.8)
            leaf['A'].add_(0.01)
        c['ids'].copy_(torch.randint(-1, 3, (300,), device='cuda'))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), k


def test_capture_beside_a_living_eager_pass_is_refused(monkeypatch):
    """The check itself, without a capture: a pass over the same leaves on the default stream is alive, then it is not."""
    c = _case(8, 64, 48, 4, 2, 'mixed', torch.float32, 0)
    leaf = {k: c[k].clone().requires_grad_(True) for k in ('A', 'B')}
    y = adapters.adapted_linear(**{**c, **leaf})
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='still alive'):
        adapters.adapted_linear(**{**c, **leaf})
    del y
    adapters.adapted_linear(**{**c, **leaf}).sum().backward()
    monkeypatch.undo()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = adapters.adapted_linear(**{**c, **leaf})
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    adapters.adapted_linear(**{**c, **leaf})
    torch.cuda.current_stream().wait_stream(side)


# ---- the model's heads ----------------------------------------------------------------------------------------------------------
def _model(layers=18):
    cfg = H.get_humaniflow_cfg_defaults()
    cfg.MODEL.NUM_RESNET_LAYERS = layers
    return init_model_for_tests(H.HumaniflowModel(torch.device('cpu'), cfg.MODEL, H.SMPL_PARENTS), seed=1).cuda().eval()


def test_model_serves_mixed_adapters():
    """A batch of requests with different adapters gives each image what a model with that adapter folded into its heads gives it (W + s B A, in 64 bits, rounded once:
    1e-5 of the values through fc1 + ELU and the small heads); ids None and untrained adapters give the plain model's outputs."""
    model = _model()
    feats = torch.randn(9, 512, device='cuda')
    with torch.no_grad():
        plain = model(None, input_feats=feats, num_samples=0)
        ad = H.LowRankAdapters(model, 3, 4, alpha=6)
        model.attach_adapters(ad)
        same = model(None, input_feats=feats, num_samples=0)
        assert all(torch.equal(plain[k], same[k]) for k in ('cam_wp', 'glob_rotmat', 'shape_mode', 'shape_log_std'))
        ids = torch.tensor([0, 1, 2, -1, 2, 1, 0, -1, 2], device='cuda')
        zero = model(None, input_feats=feats, adapter_ids=ids)
        for k in ('cam_wp', 'glob_rotmat', 'shape_mode', 'shape_log_std'):
            assert (zero[k] - plain[k]).abs().max().item() < 1e-5 * plain[k].abs().max().item() + 1e-6
        for name in ad.layers:
            getattr(ad, name + '_B').normal_(0, 0.05)
        out = model(None, input_feats=feats, adapter_ids=ids, num_samples=2)
        model.attach_adapters(None)
        for l in range(-1, 3):
            folded = _model()
            if l >= 0:
                for name in ad.layers:
                    lin = getattr(folded, name)
                    lin.weight.copy_((lin.weight.double() + 1.5 * getattr(ad, name + '_B')[l].double() @ getattr(ad, name + '_A')[l].double()).float())
            ref = folded(None, input_feats=feats)
            rows = ids == l
            for k in ('cam_wp', 'glob_rotmat', 'shape_mode', 'shape_log_std'):
                assert (out[k][rows] - ref[k][rows]).abs().max().item() < 2e-5 * max(1.0, ref[k].abs().max().item()), (k, l)


@pytest.mark.parametrize('checkpoint', [None, 'int8'])
def test_model_fits_adapters(checkpoint):
    """One training pass of the adapters alone: the encoder and the heads stay, the adapters in use get gradients, the others zeros; gradients as through nn.Linear with
    the product W + s B A of each row written out (within 1e-4; with inputs kept in 8 bits the A gradients within 3 %: 0.95 % of rounding for each kept value at most)."""
    model = _model()
    for p in model.parameters():
        p.requires_grad_(False)
    ad = H.LowRankAdapters(model, 4, 4, checkpoint=checkpoint)
    with torch.no_grad():
        for name in ad.layers:
            getattr(ad, name + '_B').normal_(0, 0.05)
    model.attach_adapters(ad)
    model.train()
    feats = torch.randn(12, 512, device='cuda')
    ids = torch.tensor([0, 1, 3, -1, 3, 1, 0, -1, 3, 0, 0, 1], device='cuda')
    wc, wm = torch.randn(12, 3, device='cuda'), torch.randn(12, 10, device='cuda')
    out = model(None, input_feats=feats, adapter_ids=ids, compute_point_est=False)
    ((out['cam_wp'] * wc).sum() + (out['shape_mode'] * wm).sum() + out['shape_log_std'].sum()).backward()
    got = {n: p.grad.double() for n, p in ad.named_parameters() if p.grad is not None}
    dbl = {n: p.detach().double().requires_grad_(True) for n, p in ad.named_parameters()}

    def lin(name, x):
        m = getattr(model, name)
        y = x @ m.weight.double().t() + m.bias.double()
        on = (ids >= 0).double()[:, None]
        l = ids.clamp(min=0)
        return y + on * torch.matmul(dbl[name + '_B'][l], torch.matmul(dbl[name + '_A'][l], x[:, :, None]))[:, :, 0]
    x = torch.nn.functional.elu(lin('fc1', feats.double()))
    sp = lin('fc_shape', x)
    ((lin('fc_cam', x) * wc).sum() + (sp[:, :10] * wm).sum() + sp[:, 10:].sum()).backward()
    for n, g in got.items():
        if n.startswith('fc_glob'):
            continue                                                     # not in this loss
        ref = dbl[n].grad
        tol = 0.03 if checkpoint and n.endswith('_A') else 1e-4
        assert (g - ref).norm().item() <= tol * ref.norm().item(), n
        assert not g[2].any()
    assert all(p.grad is None for n, p in model.named_parameters() if not n.startswith('adapters.'))


def test_fitting_adapters_with_the_encoder_in_8_bits():
    """The set as it is used: encoder trained with 8-bit checkpoints under heads with adapters, several steps, everything finite and moving."""
    model = _model()
    for name in ('fc1', 'fc_cam', 'fc_glob', 'fc_shape'):
        getattr(model, name).requires_grad_(False)
    model.attach_adapters(H.LowRankAdapters(model, 2, 4, checkpoint='int8'))
    model.image_encoder.activation_checkpoint = 'int8'
    model.train()
    opt = torch.optim.SGD([p for n, p in model.named_parameters() if n.startswith(('adapters.', 'image_encoder.'))], lr=1e-3)
    x, ids = torch.randn(4, 18, 64, 64, device='cuda'), torch.tensor([0, 1, -1, 0], device='cuda')
    before = model.adapters.fc1_B.detach().clone()
    for _ in range(3):
        opt.zero_grad()
        out = model(x, adapter_ids=ids, compute_point_est=False)
        (out['cam_wp'].square().sum() + out['shape_mode'].square().sum()).backward()
        assert all(torch.isfinite(p.grad).all() for p in model.adapters.parameters() if p.grad is not None)
        assert all(torch.isfinite(p.grad).all() for p in model.image_encoder.parameters())
        opt.step()
    assert not torch.equal(before, model.adapters.fc1_B)


def test_model_refusals():
    model = _model()
    feats = torch.randn(3, 512, device='cuda')
    ids = torch.zeros(3, dtype=torch.int32, device='cuda')
    with pytest.raises(RuntimeError, match='no adapters'):
        model(None, input_feats=feats, adapter_ids=ids)
    model.attach_adapters(H.LowRankAdapters(model, 2, 4))
    with torch.no_grad(), pytest.raises(ValueError, match='ids'):
        model(None, input_feats=feats, adapter_ids=ids[:2])
    with pytest.raises(RuntimeError, match='fixed projection'):
        model.train()(None, input_feats=feats, adapter_ids=ids)


def test_predict_takes_each_images_adapter():
    from humaniflow_amd.predict import predict_humaniflow
    model = _model()
    ad = H.LowRankAdapters(model, 2, 4)
    with torch.no_grad():
        ad.fc1_B.normal_(0, 0.05)
        ad.fc_shape_B.normal_(0, 0.05)
    model.attach_adapters(ad)
    smpl = H.SMPL(model_data=H.synthetic_smpl_model(seed=0), create_transl=False).cuda()
    x, ids = torch.randn(3, 18, 64, 64, device='cuda'), torch.tensor([1, -1, 0], device='cuda')
    res = predict_humaniflow(model, smpl, x, ['a', 'b', 'c'], num_pred_samples=0, adapter_ids=ids)
    plain = predict_humaniflow(model, smpl, x, ['a', 'b', 'c'], num_pred_samples=0)
    with torch.no_grad():
        for i in range(3):
            ref = model(x[i:i + 1], adapter_ids=ids[i:i + 1])
            assert torch.equal(res[i]['pred']['shape_mode'], ref['shape_mode'])
            same = (res[i]['pred']['shape_mode'] - plain[i]['pred']['shape_mode']).abs().max().item() < 1e-5
            assert same == (i == 1)


def test_training_step_fits_adapters():
    """train.train_step with adapter_ids: the heads' adapters and the encoder (8-bit checkpoints) move, the shared heads do not, adapters nobody used keep their values."""
    from humaniflow_amd import train as T
    from humaniflow_amd.synthetic import init_benchmark_weights
    cfg = H.get_humaniflow_cfg_defaults()
    model = init_benchmark_weights(H.HumaniflowModel(torch.device('cpu'), cfg.MODEL, H.SMPL_PARENTS), seed=0).cuda()
    for name in ('fc1', 'fc_cam', 'fc_glob', 'fc_shape'):
        getattr(model, name).requires_grad_(False)
    model.attach_adapters(H.LowRankAdapters(model, 3, 4, checkpoint='int8'))
    model.image_encoder.activation_checkpoint = 'int8'
    model.train()
    smpl = H.SMPL(model_data=H.synthetic_smpl_model(seed=0), batch_size=4, create_transl=False).cuda()
    for p in smpl.parameters():
        p.requires_grad_(False)
    params = [p for p in model.parameters() if p.requires_grad]
    opt = torch.optim.SGD(params, lr=1e-4)
    red = T.GradBucketReducer(params, None)
    batch = T.synthetic_train_batch(smpl, 4, 128, torch.device('cuda'), seed=1, data_cfg=cfg.DATA)
    ids = torch.tensor([0, 1, -1, 0], device='cuda')
    crit = H.HumaniflowLoss(cfg.LOSS, 128)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for _ in range(2):
        loss, skipped = T.train_step(model, smpl, crit, opt, red, *batch, 2, adapter_ids=ids)
        assert torch.isfinite(loss) and not skipped
    moved = {n for n, p in model.named_parameters() if not torch.equal(before[n], p)}
    assert {'adapters.fc1_B', 'adapters.fc_shape_B', 'adapters.fc1_A', 'image_encoder.conv1.weight'} <= moved
    assert not moved & {'fc1.weight', 'fc1.bias', 'fc_cam.weight', 'fc_glob.weight', 'fc_shape.weight'}
    assert torch.equal(before['adapters.fc1_B'][2], model.adapters.fc1_B[2]) and torch.equal(before['adapters.fc1_A'][2], model.adapters.fc1_A[2])


@pytest.mark.parametrize('M', [7, 300])
def test_gradient_of_a_broadcast_input_and_of_shared_adapters(M):
    """One row used by every request, and one pair of adapters used by two layers: the gradients add up."""
    c = _case(M, 64, 64, 4, 3, 'mixed', torch.float32, 8)
    row = c['x'][:1].clone().requires_grad_(True)
    A, B = c['A'].clone().requires_grad_(True), c['B'].clone().requires_grad_(True)
    args = (c['weight'], c['bias'], A, B, c['scale'], c['ids'])
    h = adapters.adapted_linear(row.expand(M, 64), *args)
    adapters.adapted_linear(h, *args).sum().backward()
    d = [t.detach().double().requires_grad_(True) for t in (c['x'][:1], A, B)]
    on, l = (c['ids'] >= 0).double()[:, None], c['ids'].clamp(min=0).long()
    f = lambda v: v @ c['weight'].double().t() + c['bias'].double() + on * c['scale'].double()[l][:, None] * torch.matmul(d[2][l], torch.matmul(d[1][l], v[:, :, None]))[:, :, 0]
    f(f(d[0].expand(M, 64))).sum().backward()
    for got, ref in zip((row, A, B), d):                                  # sums of up to 300 rows of 64-term products in 32 bits: 1e-5 of the norm is 40 times their walk
        assert (got.grad.double() - ref.grad).norm().item() <= 1e-5 * ref.grad.norm().item()
