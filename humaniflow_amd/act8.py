"""8-bit activation checkpoints: what a training step keeps of its activations between forward and backward, in 1.03 bytes per element instead of 4.

    ck = pack(x)                                       rows (M, C) float32 / bfloat16 -> Act8 (codes int8, one exponent per 32 rows of a column)
    x = unpack(ck)                                     the values that the codes stand for
    out, ck, bits, ck_out = bn_apply(y, scale, shift, residual=, relu=, keep_out=)      BatchNorm affine + identity + ReLU that leaves its checkpoint
    x = restore_activation(ck, scale, shift, bits)     the activation behind such a unit (without identity), for the next layer's weight gradient
    gy, gz, g_gamma, g_beta = bn_backward(g, ck, bits, mean, rstd, gamma, want_gz=)     BatchNorm + ReLU backward from the checkpoint

A code is x / step rounded to nearest even, step a power of two for each block of 32 consecutive rows of a column: |x - value| <= step / 2, between
1 / 254 and 1 / 127 of the block's largest magnitude.  The ReLU's mask is kept exactly (`bits`, one bit per element).  Values that are not finite come back
as NaN.  The encoder's training graph uses these when `ResNetEncoder.activation_checkpoint = 'int8'` (encoder_train.py); the adapters' backward pass takes
an Act8 in the place of its input (adapters.py).  Layouts and kernels: csrc/act8.hip.
"""
import torch

from . import _lib

BLOCK = 32                      # rows that share an exponent

MAX_ROWS = 0x7fffff00           # rows and columns are 32-bit numbers below

_DTYPES = (torch.float32, torch.bfloat16)


def _fits(M, C):
    if M > MAX_ROWS or C > MAX_ROWS:
        raise ValueError('humaniflow_amd: (%d, %d) rows: row and column numbers are 32-bit' % (M, C))


class Act8:
    """Checkpoint of rows (M, C): codes int8 (M, C), exps uint8 (ceil(M / 32), C), both contiguous (pack() and bn_apply() lay them in one buffer)."""
    __slots__ = ('shape', 'device', 'codes_ptr', 'exps_ptr', '_codes', '_exps', '_buf', '_at')

    def __init__(self, codes, exps):
        if codes.dtype != torch.int8 or exps.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError('humaniflow_amd: Act8 takes codes int8 (M, C) and exps uint8 (ceil(M / 32), C), got %s %s and %s' % (codes.dtype, tuple(codes.shape), exps.dtype))
        M, C = codes.shape
        if tuple(exps.shape) != ((M + BLOCK - 1) // BLOCK, C) or exps.device != codes.device:
            raise ValueError('humaniflow_amd: Act8: exps %s on %s do not fit codes %s on %s' % (tuple(exps.shape), exps.device, tuple(codes.shape), codes.device))
        if not (codes.is_contiguous() and exps.is_contiguous()):
            raise ValueError('humaniflow_amd: Act8 codes and exps must be contiguous')
        _fits(M, C)
        self.shape, self.device, self._codes, self._exps, self._buf = codes.shape, codes.device, codes, exps, None
        self.codes_ptr, self.exps_ptr = codes.data_ptr(), exps.data_ptr()

    @property
    def codes(self):
        if self._codes is None:
            M, C = self.shape
            self._codes = self._buf[self._at:self._at + M * C].view(torch.int8).view(M, C)
        return self._codes

    @property
    def exps(self):
        if self._exps is None:
            M, C = self.shape
            at, nb = self._at + _round16(M * C), (M + BLOCK - 1) // BLOCK
            self._exps = self._buf[at:at + nb * C].view(nb, C)
        return self._exps

    def nbytes(self):
        M, C = self.shape
        return M * C + (M + BLOCK - 1) // BLOCK * C


def _round16(n):
    return (n + 15) & ~15


def _bytes_of(M, C):
    return _round16(M * C) + _round16((M + BLOCK - 1) // BLOCK * C)


def _in_buffer(buf, at, shape, device):
    """The checkpoint of rows of `shape` whose codes and exponents lie (or will lie) at byte `at` of buf."""
    ck = Act8.__new__(Act8)
    ck.shape, ck.device, ck._codes, ck._exps, ck._buf, ck._at = shape, device, None, None, buf, at
    ck.codes_ptr = buf.data_ptr() + at
    ck.exps_ptr = ck.codes_ptr + _round16(shape[0] * shape[1])
    return ck


def _on_gpu(ck):
    if ck.device.type != 'cuda':
        _lib.require_cuda(ck.codes, 'codes')


def _rows(t, name, C=None, M=None):
    """A contiguous float32 (M, C) device tensor, or an error that names it."""
    if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or (C is not None and t.shape[1] != C) or (M is not None and t.shape[0] != M):
        raise ValueError('humaniflow_amd: `%s` must be contiguous float32 rows%s, got %s %s' % (name, '' if C is None else ' (%d, %d)' % (M, C), t.dtype, tuple(t.shape)))
    _lib.require_cuda(t, name)
    _fits(*t.shape)


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError('humaniflow_amd: `%s` is on %s, the other operands on %s' % (name, t.device, dev))


def _channels(C, *named):
    if C % 64 or C == 0:
        raise ValueError('humaniflow_amd: the BatchNorm kernels are built for multiples of 64 channels, got %d' % C)
    for name, v in named:
        if v.dtype != torch.float32 or v.shape != (C,) or not v.is_contiguous():
            raise ValueError('humaniflow_amd: `%s` must be a contiguous float32 vector of %d channels, got %s %s' % (name, C, v.dtype, tuple(v.shape)))


def _check_bits(bits, M, C):
    if bits is not None and (bits.dtype != torch.int32 or bits.shape != ((M + BLOCK - 1) // BLOCK, C) or not bits.is_contiguous()):
        raise ValueError('humaniflow_amd: `bits` must be contiguous int32 (%d, %d), got %s %s' % ((M + BLOCK - 1) // BLOCK, C, bits.dtype, tuple(bits.shape)))


def pack(x):
    """Checkpoint of x (M, C), float32 or bfloat16; rows may be strided (a view of wider rows), columns consecutive."""
    if not x.is_cuda:
        _lib.require_cuda(x, 'x')
    if x.dtype not in _DTYPES or x.dim() != 2:
        raise ValueError('humaniflow_amd: act8.pack takes float32 or bfloat16 rows (M, C), got %s %s' % (x.dtype, tuple(x.shape)))
    dev = x.device
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return pack(x)
    M, C = x.shape
    _fits(M, C)
    ld = C
    if not x.is_contiguous():
        if (C > 1 and x.stride(1) != 1) or (M > 1 and x.stride(0) < C):
            x = x.detach().contiguous()
        elif M > 1:
            ld = x.stride(0)
    ck = _in_buffer(torch.empty(_bytes_of(M, C), dtype=torch.uint8, device=dev), 0, x.shape, dev)
    _lib.check(_lib.load().hmf_act8_pack(x.data_ptr(), ld, int(x.dtype == torch.bfloat16), M, C, ck.codes_ptr, ck.exps_ptr, st), 'hmf_act8_pack')
    return ck


def unpack(ck, dtype=torch.float32):
    """The values of a checkpoint as contiguous rows (M, C), float32 or bfloat16 (a code has 7 bits: exact in both)."""
    if dtype not in _DTYPES:
        raise ValueError('humaniflow_amd: act8.unpack gives float32 or bfloat16, not %s' % dtype)
    _on_gpu(ck)
    st = _lib.stream_here(ck.device)
    if st is None:
        with torch.cuda.device(ck.device):
            return unpack(ck, dtype)
    M, C = ck.shape
    x = torch.empty(ck.shape, dtype=dtype, device=ck.device)
    _lib.check(_lib.load().hmf_act8_unpack(ck.codes_ptr, ck.exps_ptr, M, C, x.data_ptr(), int(dtype == torch.bfloat16), st), 'hmf_act8_unpack')
    return x


def bn_apply(y, scale, shift, residual=None, relu=True, keep_out=False):
    """out = relu?(y * scale + shift (+ residual)) on rows (M, C), with the checkpoint of y, the ReLU's bits (None without relu) and, with keep_out, the
    checkpoint of out: (out, ck, bits, ck_out).  C a multiple of 64, M >= 1."""
    _rows(y, 'y')
    M, C = y.shape
    _channels(C, ('scale', scale), ('shift', shift))
    if residual is not None:
        _rows(residual, 'residual', C, M)
    dev = y.device
    if scale.device != dev or shift.device != dev or (residual is not None and residual.device != dev):
        _same_device(dev, scale=scale, shift=shift, residual=residual)
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return bn_apply(y, scale, shift, residual, relu, keep_out)
    out = torch.empty_like(y)
    n = _bytes_of(M, C)
    buf = torch.empty(2 * n if keep_out else n, dtype=torch.uint8, device=dev)
    ck, ck_out = _in_buffer(buf, 0, y.shape, dev), _in_buffer(buf, n, y.shape, dev) if keep_out else None
    bits = torch.empty(((M + BLOCK - 1) // BLOCK, C), dtype=torch.int32, device=dev) if relu else None
    _lib.check(_lib.load().hmf_bn_apply_act8(y.data_ptr(), scale.data_ptr(), shift.data_ptr(), None if residual is None else residual.data_ptr(), out.data_ptr(),
                                             ck.codes_ptr, ck.exps_ptr, None if bits is None else bits.data_ptr(), ck_out.codes_ptr if keep_out else None,
                                             ck_out.exps_ptr if keep_out else None, M, C, int(relu), st), 'hmf_bn_apply_act8')
    return out, ck, bits, ck_out


def restore_activation(ck, scale, shift, bits=None):
    """The float32 output of a bn_apply without residual, from its checkpoint: relu(value * scale + shift), zero where the ReLU's bit is clear (bits None:
    the affine alone)."""
    _on_gpu(ck)
    M, C = ck.shape
    _channels(C, ('scale', scale), ('shift', shift))
    _check_bits(bits, M, C)
    dev = ck.device
    if scale.device != dev or shift.device != dev or (bits is not None and bits.device != dev):
        _same_device(dev, scale=scale, shift=shift, bits=bits)
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return restore_activation(ck, scale, shift, bits)
    x = torch.empty(ck.shape, dtype=torch.float32, device=dev)
    _lib.check(_lib.load().hmf_act8_restore_activation(ck.codes_ptr, ck.exps_ptr, None if bits is None else bits.data_ptr(), scale.data_ptr(), shift.data_ptr(),
                                                       x.data_ptr(), M, C, st), 'hmf_act8_restore_activation')
    return x


def bn_backward(g, ck, bits, mean, rstd, gamma, want_gz=False):
    """g = dL/d out of a bn_apply (M, C) -> (gy = dL/dy, gz = the masked gradient or None, dL/d gamma, dL/d beta); bits None: no ReLU."""
    _rows(g, 'g')
    M, C = g.shape
    _channels(C, ('mean', mean), ('rstd', rstd), ('gamma', gamma))
    if ck.shape != g.shape:
        raise ValueError('humaniflow_amd: the checkpoint holds %s rows, the gradient is %s' % (tuple(ck.shape), (M, C)))
    _check_bits(bits, M, C)
    dev = g.device
    if ck.device != dev or mean.device != dev or rstd.device != dev or gamma.device != dev or (bits is not None and bits.device != dev):
        _same_device(dev, checkpoint=ck, bits=bits, mean=mean, rstd=rstd, gamma=gamma)
    st = _lib.stream_here(dev)
    if st is None:
        with torch.cuda.device(dev):
            return bn_backward(g, ck, bits, mean, rstd, gamma, want_gz)
    gy = torch.empty_like(g)
    gz = torch.empty_like(g) if want_gz else None
    gg, gb = torch.empty_like(gamma), torch.empty_like(gamma)
    lib = _lib.load()
    n = lib.hmf_bn_backward_act8_workspace_bytes(M, C)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.hmf_bn_backward_act8(g.data_ptr(), ck.codes_ptr, ck.exps_ptr, None if bits is None else bits.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                        gamma.data_ptr(), gy.data_ptr(), None if gz is None else gz.data_ptr(), gg.data_ptr(), gb.data_ptr(), M, C, ws.data_ptr(), n,
                                        st), 'hmf_bn_backward_act8')
    return gy, gz, gg, gb
