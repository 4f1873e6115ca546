"""Cases of the operators for fitting a trained model to new subjects: activation checkpoints in 8 bits (the encoder's training graph) and low-rank
adapters of many requests beside a shared projection (the heads), with their plain forms in torch operators and their definitions in 64 bits.

An 8-bit checkpoint of rows (M, C) is: codes int8 (M, C); exps uint8 (ceil(M / 32), C), one biased exponent E per 32 rows of a column; the value is
code * 2^(E - 133).  E = exponent field of the block's largest finite magnitude, one more where that would round to 128 steps, within [7, 254]; a code
is the value over the step rounded to nearest even; -128 stands for a value that is not finite.  ReLU bits: uint32 words held as int32
(ceil(M / 32), C), bit i of word t = row 32 t + i.
"""
import math

import torch

own = False
LOW = -126.0                 # exponent of the smallest step


def _case(op, name=None, **k):
    c = dict(op=op, **k)
    return dict(c, name=name) if name else c


def listed():
    return [
        # image features of a fine-tuning batch kept for the heads' backward: few rows, an odd width, a row pitch
        _case('pack', 'pack_features_odd', M=72, C=515, pad=13, dtype='float32'),
        # a long batch of 16-bit rows
        _case('pack', 'pack_rows_bf16', M=8192, C=2048, pad=0, dtype='bfloat16'),
        # last block of the 18-layer encoder at the training batch of 72 images: 8 x 8 maps, identity added
        _case('save', 'save_layer4', M=4608, C=512, residual=True),
        # the largest maps behind the stem of the 50-layer encoder at the training batch: 64 x 64, identity added
        _case('save', 'save_layer1_wide', M=294912, C=256, residual=True),
        # inner unit of the 18-layer encoder: its activation is rebuilt from the checkpoint for the next layer's weight gradient
        _case('save', 'save_layer2_inner', M=73728, C=128, residual=False),
        _case('bn_back', 'bn_back_layer4', M=4608, C=512, gz=False),
        _case('bn_back', 'bn_back_layer1_wide', M=294912, C=256, gz=True),
        # one image through fc1 of the 50-layer model with one adapter: the predict shape
        _case('adapt', 'adapt_one_image', M=1, K=2048, N=1024, r=16, L=1, ids='one', dtype='float32'),
        # the shape head of a batch of 32 images of as many subjects: 20 outputs
        _case('adapt', 'adapt_shape_head', M=32, K=1024, N=20, r=4, L=32, ids='mixed', dtype='float32'),
        # a long batch of requests' rows in 16 bits
        _case('adapt', 'adapt_rows_bf16', M=4096, K=2048, N=1024, r=16, L=16, ids='runs', dtype='bfloat16'),
        # fc1 of the 18-layer model at the training batch
        _case('adapt_back', 'adapt_back_fc1', M=72, K=512, N=512, r=8, L=12, ids='mixed', dtype='float32', x8=False),
        # a long batch whose inputs were kept in 8 bits
        _case('adapt_back', 'adapt_back_rows8', M=4096, K=2048, N=1024, r=16, L=16, ids='mixed', dtype='bfloat16', x8=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['pack', 'save', 'bn_back', 'adapt', 'adapt_back'])
    if op == 'pack':
        C = _log(rng, 1, 2048)
        M = _log(rng, 8, 16384)
        return _case(op, M=M, C=C, pad=rng.choice([0, 0, 4, rng.randrange(1, 40)]), dtype=rng.choice(['float32', 'bfloat16']))
    if op in ('save', 'bn_back'):
        C = 64 * _log(rng, 1, 32)
        M = min(_log(rng, 40, 294912), 75000000 // C)
        return _case(op, M=M, C=C, **({'residual': rng.random() < 0.5} if op == 'save' else {'gz': rng.random() < 0.5}))
    c = dict(M=_log(rng, 1, 4096), K=_log(rng, 32, 2048), N=_log(rng, 3, 2048), r=_log(rng, 1, 64), L=_log(rng, 1, 64),
             ids=rng.choice(['one', 'runs', 'mixed']), dtype=rng.choice(['float32', 'bfloat16']))
    if rng.random() < 0.6:
        c['K'] = max(32, c['K'] // 32 * 32)
    if op == 'adapt_back':
        c['x8'] = rng.random() < 0.5
    return _case(op, **c)


def _pack(x):
    """Plain 8-bit checkpoint of x (M, C)."""
    M, C = x.shape
    nb = (M + 31) // 32
    x = x.float()
    fine = torch.isfinite(x)
    v = torch.where(fine, x, torch.zeros_like(x))
    v = torch.cat([v, v.new_zeros(nb * 32 - M, C)]).view(nb, 32, C)
    top = v.abs().amax(dim=1)
    E = ((top.contiguous().view(torch.int32) + 0x10000) >> 23).clamp(7, 254)
    inv = ((266 - E - 6) << 23).view(torch.float32)                       # 2^(133 - E) = exponent field 260 - E, a normal number for E >= 7
    q = torch.round(v * inv[:, None]).clamp(-127, 127).view(nb * 32, C)[:M]
    codes = torch.where(fine, q, torch.full_like(q, -128.0)).to(torch.int8)
    return codes, E.to(torch.uint8)


def _unpack(codes, exps):
    """The values that the codes stand for, in 32 bits."""
    M, C = codes.shape
    step = torch.ldexp(torch.ones((), device=codes.device, dtype=torch.float64), exps.to(torch.int32) - 133).float()
    v = codes.float() * step.repeat_interleave(32, dim=0)[:M]
    return torch.where(codes == -128, torch.full_like(v, float('nan')), v)


def _bits(words, M):
    i = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[:, None, :] >> i[None, :, None]) & 1).view(-1, words.shape[1])[:M].bool()


def _words(on):
    M, C = on.shape
    nb = (M + 31) // 32
    p = torch.cat([on, on.new_zeros(nb * 32 - M, C)]).view(nb, 32, C).long()
    w = (p << torch.arange(32, device=on.device)[None, :, None]).sum(dim=1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)
    op, M = case['op'], case['M']
    s = {'case': case}
    if op == 'pack':
        x = (rn(M, case['C'] + case['pad']) * torch.exp(rn(case['C'] + case['pad']))).to(getattr(torch, case['dtype']))
        s['x'] = x[:, :case['C']]
        return s
    if op in ('save', 'bn_back'):
        C = case['C']
        y = rn(M, C) * torch.exp(0.5 * rn(C)) + 0.5 * rn(C)                # a convolution's output: a scale and a mean for each channel
        mean = y.mean(dim=0)
        rstd = torch.rsqrt(y.var(dim=0, unbiased=False) + 1e-5)
        s['gamma'] = 1.0 + 0.2 * rn(C)
        if op == 'save':
            s['y'], s['scale'] = y, s['gamma'] * rstd
            s['shift'] = 0.1 * rn(C) - mean * s['scale']
            s['residual'] = rn(M, C).relu() if case['residual'] else None
            return s
        s['mean'], s['rstd'] = mean, rstd
        s['codes'], s['exps'] = _pack(y)
        s['bits'] = _words(rn(M, C) > 0)
        s['g'] = 1e-3 * rn(M, C) * torch.exp(0.5 * rn(C))
        return s
    K, N, r, L = (case[k] for k in 'KNrL')
    dt = getattr(torch, case['dtype'])
    s['x'] = rn(M, K).to(dt)
    s['weight'], s['bias'] = (rn(N, K) / K ** 0.5).to(dt), (0.1 * rn(N)).to(dt)
    s['A'], s['B'] = (rn(L, r, K) / K ** 0.5).to(dt), (0.3 * rn(L, N, r) / r ** 0.5).to(dt)
    s['scale'] = 0.5 + torch.rand(L, device=dev, generator=g)
    if case['ids'] == 'one':
        ids = torch.zeros(M, dtype=torch.int32, device=dev)
    elif case['ids'] == 'mixed':                                          # every row a request of its own, some without an adapter
        ids = torch.randint(-1, L, (M,), device=dev, generator=g, dtype=torch.int32)
    else:                                                                 # requests of many rows, one behind the other
        cuts = torch.sort(torch.randint(0, M + 1, (max(1, min(M, 2 * L)) - 1,), device=dev, generator=g)).values
        run_of = torch.searchsorted(cuts, torch.arange(M, device=dev), right=True)
        ids = torch.randint(-1, L, (2 * L + M,), device=dev, generator=g, dtype=torch.int32)[run_of]
    s['ids'] = ids
    if op == 'adapt_back':
        s['dy'] = (1e-2 * rn(M, N)).to(dt)
        if case['x8']:
            s['codes'], s['exps'] = _pack(s['x'])
            s['x'] = None
        x = s['x'].float() if s['x'] is not None else _unpack(s['codes'], s['exps'])
        s['t'] = _low(x, s['A'].float(), s['scale'], ids)                   # kept by the forward pass
    return s


def _pick(ids, L):
    """(M, L) of 0 / 1: which adapter a row uses."""
    return (ids[:, None] == torch.arange(L, device=ids.device, dtype=ids.dtype)[None]).float()


def _low(x, A, scale, ids):
    """s (x A_l^T) with the row's own adapter l, zero without one: (M, r)."""
    L, r, K = A.shape
    all_ = (x @ A.reshape(L * r, K).t()).view(-1, L, r)
    return (all_ * (_pick(ids, L) * scale)[:, :, None]).sum(dim=1)


def _spread(t, ids, L):
    """(M, L r): t in the columns of the row's own adapter, zero elsewhere."""
    return (t[:, None, :] * _pick(ids, L)[:, :, None]).reshape(t.shape[0], -1)


def run(state):
    case = state['case']
    op = case['op']
    if own:
        from humaniflow_amd import act8, adapters
        if op == 'pack':
            return act8.unpack(act8.pack(state['x']))
        if op == 'save':
            out, ck, bits, ck_out = act8.bn_apply(state['y'], state['scale'], state['shift'], residual=state['residual'], relu=True, keep_out=case['residual'])
            x = act8.unpack(ck_out) if case['residual'] else act8.restore_activation(ck, state['scale'], state['shift'], bits)
            return {'out': out, 'x': x}
        if op == 'bn_back':
            gy, gz, gg, gb = act8.bn_backward(state['g'], act8.Act8(state['codes'], state['exps']), state['bits'], state['mean'], state['rstd'],
                                              state['gamma'], want_gz=case['gz'])
            return {'gy': gy, 'gz': gz, 'g_gamma': gg, 'g_beta': gb}
        if op == 'adapt':
            return adapters.adapted_linear(state['x'], state['weight'], state['bias'], state['A'], state['B'], state['scale'], state['ids'])
        x = act8.Act8(state['codes'], state['exps']) if case['x8'] else state['x']
        dx, dA, dB = adapters.adapted_linear_backward(state['dy'], x, state['t'], state['weight'], state['A'], state['B'], state['scale'], state['ids'])
        return {'dx': dx, 'dA': dA, 'dB': dB}
    if op == 'pack':
        return _unpack(*_pack(state['x']))
    if op == 'save':
        y, res = state['y'], state['residual']
        scale, shift = state['scale'].double(), state['shift'].double()
        v = (y.double() * scale + shift).float()                          # one rounding: values next to zero decide a bit
        if res is not None:
            v = v + res
        out = v.relu()
        if res is not None:
            return {'out': out, 'x': _unpack(*_pack(out))}
        words = _words(v > 0)
        x = (_unpack(*_pack(y)) * state['scale'] + state['shift']).relu()
        return {'out': out, 'x': torch.where(_bits(words, y.shape[0]), x, torch.zeros_like(x))}
    if op == 'bn_back':
        M = case['M']
        xhat = (_unpack(state['codes'], state['exps']) - state['mean']) * state['rstd']
        gz = torch.where(_bits(state['bits'], M), state['g'], torch.zeros_like(state['g']))
        sg, sgx = gz.double().sum(dim=0), (gz * xhat).double().sum(dim=0)
        gy = state['gamma'] * state['rstd'] * (gz - (sg / M).float() - xhat * (sgx / M).float())
        return {'gy': gy, 'gz': gz if case['gz'] else None, 'g_gamma': sgx.float(), 'g_beta': sg.float()}
    ids, scale = state['ids'], state['scale']
    A, B, W = state['A'].float(), state['B'].float(), state['weight'].float()
    L, r, K = A.shape
    N = W.shape[0]
    if op == 'adapt':
        x = state['x'].float()
        wide = _spread(_low(x, A, scale, ids), ids, L)
        y = x @ W.t() + state['bias'].float() + wide @ B.transpose(0, 1).reshape(N, L * r).t()
        return y.to(state['x'].dtype)
    x = _unpack(state['codes'], state['exps']) if case['x8'] else state['x'].float()
    dy = state['dy'].float()
    M = dy.shape[0]
    u = ((dy @ B.transpose(0, 1).reshape(N, L * r)).view(M, L, r) * (_pick(ids, L) * scale)[:, :, None]).reshape(M, L * r)
    dx = dy @ W + u @ A.reshape(L * r, K)
    dA = (u.t() @ x).view(L, r, K)
    dB = (_spread(state['t'], ids, L).t() @ dy).view(L, r, N).transpose(1, 2)
    dt = state['dy'].dtype
    return {'dx': dx.to(dt), 'dA': dA.to(dt), 'dB': dB.contiguous().to(dt)}


def work(case):
    """Every input read once, every output written once; the multiply-adds of the definitions."""
    op, M = case['op'], case['M']
    if op in ('pack', 'save', 'bn_back'):
        C = case['C']
        n, blocks = M * C, (M + 31) // 32 * C
        if op == 'pack':
            return {'bytes': n * (2 if case['dtype'] == 'bfloat16' else 4) + 2 * (n + blocks) + 4 * n, 'flops': 4 * n}
        if op == 'save':
            kept = n + blocks
            return {'bytes': 4 * n * (4 if case['residual'] else 3) + 8 * C + kept + 4 * blocks + (2 * kept if case['residual'] else kept + 4 * blocks),
                    'flops': 6 * n}
        return {'bytes': 4 * n + n + 5 * blocks + 4 * n * (2 if case['gz'] else 1) + 20 * C, 'flops': 10 * n}
    K, N, r, L = (case[k] for k in 'KNrL')
    z = 2 if case['dtype'] == 'bfloat16' else 4
    used = min(L, M) * r * (K + N) * z
    if op == 'adapt':
        return {'bytes': z * (M * K + N * K + N + M * N) + used + 4 * (M + L), 'flops': 2 * M * K * N + 2 * M * r * (K + N)}
    kept = M * K + (M + 31) // 32 * K if case['x8'] else z * M * K
    return {'bytes': z * (M * N + N * K + M * K) + kept + used + L * r * (K + N) * z + 4 * M * r + 4 * (M + L),
            'flops': 2 * M * K * N + 4 * M * r * (K + N)}


def _exact_values(v):
    """What an 8-bit checkpoint of v (float64 values of the input's type) stands for, column blocks of 32 rows."""
    out = torch.empty_like(v)
    whole = v.shape[0] // 32 * 32
    for part, to in ((v[:whole].view(-1, 32, v.shape[1]), out[:whole]), (v[whole:][None], out[whole:])):
        if part.numel() == 0:
            continue
        top = part.abs().amax(dim=1, keepdim=True)
        _, k = torch.frexp(top)                                           # top = m 2^k, 0.5 <= m < 1
        e = torch.where(top > 0, k.double() - 7.0, torch.full_like(top, LOW))
        e = torch.where(top * torch.exp2(-e) >= 127.5, e + 1.0, e).clamp(min=LOW)
        step = torch.exp2(e)
        to.copy_((torch.round(part / step) * step).reshape(to.shape))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'pack':
        return _exact_values(s['x'].double())
    if op == 'save':
        y, scale, shift = s['y'].double(), s['scale'].double(), s['shift'].double()
        v = y * scale + shift
        if s['residual'] is not None:
            v = v + s['residual'].double()
            out = v.clamp(min=0.0)
            return {'out': out, 'x': _exact_values(out.float().double())}  # the kept activation is the 32-bit one
        x = (_exact_values(y) * scale + shift).clamp(min=0.0)
        return {'out': v.clamp(min=0.0), 'x': x * (v > 0).double()}
    if op == 'bn_back':
        M, C = case['M'], case['C']
        row = torch.arange(M, device=s['g'].device)
        block = row // 32
        step = torch.exp2(s['exps'].double() - 133.0)
        xhat = (s['codes'].double() * step[block] - s['mean'].double()) * s['rstd'].double()
        on = ((s['bits'].long()[block] >> (row % 32)[:, None]) & 1).double()
        gz = s['g'].double() * on
        sg, sgx = gz.sum(dim=0), (gz * xhat).sum(dim=0)
        gy = s['gamma'].double() * s['rstd'].double() * (gz - sg / M - xhat * (sgx / M))
        return {'gy': gy, 'gz': gz if case['gz'] else None, 'g_gamma': sgx, 'g_beta': sg}
    ids, scale, W = s['ids'].long(), s['scale'].double(), s['weight'].double()
    if op == 'adapt':
        x = s['x'].double()
        y = x @ W.t() + s['bias'].double()
        for l in range(case['L']):
            rows = torch.nonzero(ids == l)[:, 0]
            y[rows] += scale[l] * (x[rows] @ s['A'][l].double().t()) @ s['B'][l].double().t()
        return y
    dy = s['dy'].double()
    if case['x8']:
        block = torch.arange(case['M'], device=dy.device) // 32
        x = s['codes'].double() * torch.exp2(s['exps'].double() - 133.0)[block]
    else:
        x = s['x'].double()
    dx = dy @ W
    dA, dB = torch.zeros(s['A'].shape, dtype=torch.float64, device=dy.device), torch.zeros(s['B'].shape, dtype=torch.float64, device=dy.device)
    for l in range(case['L']):
        rows = torch.nonzero(ids == l)[:, 0]
        u = scale[l] * (dy[rows] @ s['B'][l].double())
        dx[rows] += u @ s['A'][l].double()
        dA[l] = u.t() @ x[rows]
        dB[l] = dy[rows].t() @ s['t'][rows].double()
    return {'dx': dx, 'dA': dA, 'dB': dB}
