"""Low-rank adapters of many requests beside a shared projection: one trained model, a small difference to its heads for every subject, camera or data set.

    y[m] = W x[m] + b + s_l B_l A_l x[m],   l = ids[m]   (negative: no adapter)

    y = adapted_linear(x, weight, bias, A, B, scale, ids)                        differentiable w.r.t. x, A and B (the shared projection is held fixed)
    y, t = adapted_linear_forward(...);  dx, dA, dB = adapted_linear_backward(dy, x, t, weight, A, B, scale, ids)

x (M, K), weight (N, K), bias (N) or None, A (L, r, K), B (L, N, r): all float32 or all bfloat16; scale (L) float32; ids (M) int32 / int64; r <= 64,
L + M / 256 <= 65,535 and M max(K, N) up to some 1.7e10.  An id of L or more has no adapter to go with: that row's outputs
are NaN.  The backward pass takes x as it was or as an 8-bit checkpoint (act8.Act8).
`LowRankAdapters` holds the adapters of a HumaniflowModel's heads (models/humaniflow_model.py:232-252): `model.attach_adapters(...)`, then
`model(..., adapter_ids=ids)`.  Kernels: csrc/adapters.hip.
"""
import torch
from torch import nn

from . import _lib, act8
from .autograd import leaves_of, note_stream, refuse_capture_beside_default_stream_pass

MAX_RANK = 64


_TYPES = (torch.float32, torch.bfloat16)


def _check(x, weight, bias, A, B, scale, ids):
    """Shapes, types and devices (x: a tensor or an Act8) -> (M, K, N, r, L, ids as int32)."""
    dt, ws, xs, As, Bs = weight.dtype, weight.shape, x.shape, A.shape, B.shape
    if dt not in _TYPES:
        raise ValueError('humaniflow_amd: adapted_linear is built for float32 and bfloat16, got %s' % dt)
    if len(ws) != 2 or len(As) != 3 or len(Bs) != 3 or len(xs) != 2:
        raise ValueError('humaniflow_amd: adapted_linear takes x (M, K), weight (N, K), A (L, r, K), B (L, N, r); got %s, %s, %s, %s' % (tuple(xs), tuple(ws), tuple(As), tuple(Bs)))
    M, K = xs
    N, L, r = ws[0], As[0], As[1]
    if ws[1] != K or As[2] != K or Bs != (L, N, r) or L < 1 or r < 1 or K < 1 or N < 1:
        raise ValueError('humaniflow_amd: adapted_linear: x %s, weight %s, A %s, B %s do not fit' % (tuple(xs), tuple(ws), tuple(As), tuple(Bs)))
    if r > MAX_RANK:
        raise ValueError('humaniflow_amd: adapters of rank %d: built up to %d' % (r, MAX_RANK))
    if max(M, K, N, L) > act8.MAX_ROWS:
        raise ValueError('humaniflow_amd: adapted_linear: x %s, weight %s, A %s: sizes are 32-bit' % (tuple(xs), tuple(ws), tuple(As)))
    if A.dtype != dt or B.dtype != dt or (bias is not None and (bias.dtype != dt or bias.shape != (N,))):
        raise ValueError('humaniflow_amd: adapted_linear: bias (%d), A and B must have the weight\'s type %s' % (N, dt))
    if scale.dtype != torch.float32 or scale.shape != (L,):
        raise ValueError('humaniflow_amd: `scale` must be float32 (%d), got %s %s' % (L, scale.dtype, tuple(scale.shape)))
    if ids.shape != (M,) or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError('humaniflow_amd: `ids` must be int32 or int64 (%d), got %s %s' % (M, ids.dtype, tuple(ids.shape)))
    if not weight.is_cuda:
        _lib.require_cuda(weight, 'weight')
    dev, at = weight.device, weight.get_device()                             # numbers compare in half the time of devices, and this is a small call's host time
    if (x.device != dev or A.get_device() != at or B.get_device() != at or scale.get_device() != at or ids.get_device() != at
            or (bias is not None and bias.get_device() != at)):
        for name, t in (('x', x), ('bias', bias), ('A', A), ('B', B), ('scale', scale), ('ids', ids)):
            if t is not None and t.device != dev:
                raise ValueError('humaniflow_amd: `%s` is on %s, the weight on %s' % (name, t.device, dev))
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, 0x7fffffff).to(torch.int32)                  # what does not fit 32 bits stays out of range
    return M, K, N, r, L, ids if ids.is_contiguous() else ids.contiguous()


def _dense(t):
    """t, or a contiguous copy of it (only its memory is used: no graph)."""
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _rows(x):
    """x with consecutive columns (rows may have a pitch) and that pitch."""
    M, K = x.shape
    if x.is_contiguous():
        return x, K
    if (K > 1 and x.stride(1) != 1) or (M > 1 and x.stride(0) < K):
        return x.detach().contiguous(), K
    return x, x.stride(0) if M > 1 else K


def adapted_linear_forward(x, weight, bias, A, B, scale, ids, need_t=True):
    """(y (M, N), t (M, r) float32): t = s_l A_l x is what the backward pass takes (None without need_t)."""
    M, K, N, r, L, ids = _check(x, weight, bias, A, B, scale, ids)
    if x.dtype != weight.dtype:
        raise ValueError('humaniflow_amd: adapted_linear: x is %s, the weight %s' % (x.dtype, weight.dtype))
    x, ldx = _rows(x)
    if not (weight.is_contiguous() and A.is_contiguous() and B.is_contiguous() and scale.is_contiguous() and (bias is None or bias.is_contiguous())):
        weight, bias, A, B, scale = _dense(weight), _dense(bias), _dense(A), _dense(B), _dense(scale)
    dev = weight.device
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return adapted_linear_forward(x, weight, bias, A, B, scale, ids, need_t)
    y = torch.empty((M, N), dtype=weight.dtype, device=dev)
    t = torch.empty((M, r), dtype=torch.float32, device=dev) if need_t else None
    lib = _lib.load()
    bf16 = int(weight.dtype == torch.bfloat16)
    xp, wp, ap = x.data_ptr(), weight.data_ptr(), A.data_ptr()
    n = lib.hmf_adapted_linear_workspace_bytes_for(xp, ldx, wp, ap, M, K, N, r, L, bf16)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None      # a few rows need none
    _lib.check(lib.hmf_adapted_linear(xp, ldx, wp, None if bias is None else bias.data_ptr(), ap, B.data_ptr(), scale.data_ptr(), ids.data_ptr(), M, K, N, r, L, bf16, y.data_ptr(), None if t is None else t.data_ptr(), None if ws is None else ws.data_ptr(), n, st), 'hmf_adapted_linear')
    return y, t


def adapted_linear_backward(dy, x, t, weight, A, B, scale, ids, need_dx=True):
    """(dL/dx or None, dL/dA, dL/dB) from dy = dL/dy; x: the forward's input or its 8-bit checkpoint; t: what the forward returned."""
    kept8 = isinstance(x, act8.Act8)
    M, K, N, r, L, ids = _check(x, weight, None, A, B, scale, ids)
    dt, dev = weight.dtype, weight.device
    if not kept8 and x.dtype != dt:
        raise ValueError('humaniflow_amd: adapted_linear: x is %s, the weight %s' % (x.dtype, dt))
    if dy.dtype != dt or dy.shape != (M, N) or dy.device != dev:
        raise ValueError('humaniflow_amd: `dy` must be %s (%d, %d) on %s, got %s %s on %s' % (dt, M, N, dev, dy.dtype, tuple(dy.shape), dy.device))
    if t.dtype != torch.float32 or t.shape != (M, r) or t.device != dev:
        raise ValueError('humaniflow_amd: `t` must be float32 (%d, %d) on %s, got %s %s on %s' % (M, r, dev, t.dtype, tuple(t.shape), t.device))
    dy = _dense(dy)
    if dy.data_ptr() % 16:
        dy = dy.clone()
    if not (t.is_contiguous() and weight.is_contiguous() and A.is_contiguous() and B.is_contiguous() and scale.is_contiguous()):
        t, weight, A, B, scale = _dense(t), _dense(weight), _dense(A), _dense(B), _dense(scale)
    if M == 0:
        return (torch.empty((0, K), dtype=dt, device=dev) if need_dx else None), torch.zeros_like(A), torch.zeros_like(B)
    if kept8:
        xp, ldx, exps = x.codes_ptr, K, x.exps_ptr
    else:
        x, ldx = _rows(x)
        xp, exps = x.data_ptr(), None
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return adapted_linear_backward(dy, x, t, weight, A, B, scale, ids, need_dx)
    dx = torch.empty((M, K), dtype=dt, device=dev) if need_dx else None
    dA, dB = torch.empty_like(A), torch.empty_like(B)
    lib = _lib.load()
    bf16 = int(dt == torch.bfloat16)
    n = lib.hmf_adapted_linear_backward_workspace_bytes_for(M, K, N, r, L, bf16, int(need_dx))
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.hmf_adapted_linear_backward(dy.data_ptr(), xp, ldx, exps, t.data_ptr(), weight.data_ptr(), A.data_ptr(), B.data_ptr(), scale.data_ptr(), ids.data_ptr(),
                                               M, K, N, r, L, bf16, None if dx is None else dx.data_ptr(), dA.data_ptr(), dB.data_ptr(), ws.data_ptr(), n, st),
               'hmf_adapted_linear_backward')
    return dx, dA, dB


class _AdaptedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, A, B, scale, ids, checkpoint):
        y, t = adapted_linear_forward(x, weight, bias, A, B, scale, ids)
        ck = act8.pack(x) if checkpoint == 'int8' else checkpoint           # with a checkpoint x itself is not kept
        ctx.save_for_backward(x if ck is None else None, t, weight, A, B, scale, ids, *((None, None) if ck is None else (ck.codes, ck.exps)))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, t, weight, A, B, scale, ids, codes, exps = ctx.saved_tensors
        if codes is not None:
            x = act8.Act8(codes, exps)
        dx, dA, dB = adapted_linear_backward(dy, x, t, weight, A, B, scale, ids, need_dx=ctx.needs_input_grad[0])
        return dx, None, None, dA, dB, None, None, None


def adapted_linear(x, weight, bias, A, B, scale, ids, checkpoint=None):
    """y (M, N).  Differentiable w.r.t. x, A and B; the shared projection is held fixed (a weight, bias or scale that requires a gradient is refused).
    checkpoint='int8': the backward pass keeps x in 8 bits; act8.pack(x) in its place is kept as it is, so that layers which read the same x share one.  To capture forward
    and backward into a HIP graph, first let go of every eager pass over the same parameters (its outputs and loss)."""
    if isinstance(checkpoint, act8.Act8):
        if checkpoint.shape != x.shape or checkpoint.device != x.device:
            raise ValueError('humaniflow_amd: the checkpoint holds %s rows on %s, x is %s on %s' % (tuple(checkpoint.shape), checkpoint.device, tuple(x.shape), x.device))
    elif checkpoint not in (None, 'int8'):
        raise ValueError("humaniflow_amd: checkpoint must be None, 'int8' or an Act8 of x, got %r" % (checkpoint,))
    if torch.is_grad_enabled():
        if weight.requires_grad or scale.requires_grad or (bias is not None and bias.requires_grad):
            raise RuntimeError('humaniflow_amd: adapters are fitted beside a fixed projection: call requires_grad_(False) on its weight and bias, and on scale')
        if x.requires_grad or A.requires_grad or B.requires_grad:
            y = _AdaptedLinear.apply(x, weight, bias, A, B, scale, ids, checkpoint)
            leaves = leaves_of(y.grad_fn)
            note_stream(leaves, y.device)
            refuse_capture_beside_default_stream_pass(leaves, 'adapted_linear')
            return y
    return adapted_linear_forward(x, weight, bias, A, B, scale, ids, need_t=False)[0]


class LowRankAdapters(nn.Module):
    """Adapters of the heads of a HumaniflowModel: parameters `<layer>_A` (L, r, in) and `<layer>_B` (L, out, r) for each of `layers`, one shared factor
    alpha / r.  A starts as the linear layers do, B at zero: an untrained adapter changes nothing.  checkpoint='int8': fitting keeps the layers' inputs in 8 bits."""
    HEADS = ('fc1', 'fc_cam', 'fc_glob', 'fc_shape')

    def __init__(self, model, num_adapters, rank, alpha=None, layers=HEADS, checkpoint=None):
        super().__init__()
        if checkpoint not in (None, 'int8'):
            raise ValueError("humaniflow_amd: checkpoint must be None or 'int8', got %r" % (checkpoint,))
        if num_adapters < 1 or not 1 <= rank <= MAX_RANK:
            raise ValueError('humaniflow_amd: %d adapters of rank %d: at least one, of rank 1 to %d' % (num_adapters, rank, MAX_RANK))
        unknown = [n for n in layers if n not in self.HEADS]
        if unknown or not layers:
            raise ValueError('humaniflow_amd: adapters go with %s, not %s' % (', '.join(self.HEADS), unknown))
        self.num_adapters, self.rank, self.layers, self.checkpoint = num_adapters, rank, tuple(layers), checkpoint
        ref = model.fc1.weight
        self.register_buffer('scale', torch.full((num_adapters,), float(rank if alpha is None else alpha) / rank, dtype=torch.float32, device=ref.device))
        for name in self.layers:
            lin = getattr(model, name)
            A = torch.empty(num_adapters, rank, lin.in_features, dtype=torch.float32, device=ref.device).uniform_(-1, 1) / lin.in_features ** 0.5
            self.register_parameter(name + '_A', nn.Parameter(A))
            self.register_parameter(name + '_B', nn.Parameter(torch.zeros(num_adapters, lin.out_features, rank, dtype=torch.float32, device=ref.device)))

    def keep(self, x, names):
        """The 8-bit checkpoint of x that the layers `names`, which all read it, share (linear's `kept`), or None where the option is off or nothing is differentiated."""
        if self.checkpoint is None or not torch.is_grad_enabled() or not any(n in self.layers for n in names):
            return None
        return act8.pack(x) if x.requires_grad or any(p.requires_grad for p in self.parameters()) else None

    def linear(self, name, lin, x, ids, kept=None):
        """lin(x) with the rows' own adapters, or lin(x) alone for a layer that has none."""
        if name not in self.layers:
            return torch.nn.functional.linear(x, lin.weight, lin.bias)
        return adapted_linear(x, lin.weight, lin.bias, getattr(self, name + '_A'), getattr(self, name + '_B'), self.scale, ids, self.checkpoint if kept is None else kept)
