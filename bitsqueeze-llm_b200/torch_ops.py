"""PyTorch door onto the operators on microscaled 4-bit matrices, on gradients, and of the two ends of a training step (bsq_fp4_*, bsq_grad_norm_clip, bsq_linear_xent*,
bsq_orthogonalize in include/bitsqz_llm_c.h).

    x4 = fp4_quantize(x, NVFP4)                 # activations, parked in 4 bits: 0.5625 bytes an element
    w4 = fp4_quantize(w, NVFP4)
    y = fp4_matmul(x4, w4)                      # x w^T on the block-scaled tensor cores
    dx = fp4_grad_input(dy, w4)                 # dy w
    dw = fp4_grad_weight(dy, x4, torch.float32) # dy^T x, from the parked activations
    x_again = fp4_dequantize(x4, torch.bfloat16)
    norm = clip_grad_norm([dw, ...], 1.0)
    y = fp4_linear(x, w)                        # the first five under autograd
    loss = linear_cross_entropy(y, head, t)     # over a vocabulary, without its logits, under autograd
    updates = orthogonalize([dw, ...])          # Newton-Schulz steps

Calls enqueue on PyTorch's current stream of their tensors' device and return; nothing is synchronised, nothing is kept from one
call to the next, and calls may be captured in a CUDA graph.  Tensors that are used on another stream than the one they were made
on are the caller's to order, as with PyTorch's own operators.  A wait inside a product that ran out of tries leaves NaN in the result.
Every result comes from the shared library; there is no fallback.  The operators are not registered with torch.compile: a compiled graph breaks at each call, and with
fullgraph=True compilation fails there.
"""
import math
from array import array
from operator import attrgetter

import torch
from torch.autograd.forward_ad import unpack_dual

from . import MXFP4, NVFP4, lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BLOCK = {MXFP4: 32, NVFP4: 16}
_HEAD = 128
_NORM_SCRATCH = 16384                                      # bsq_grad_norm_scratch_bytes
_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice
_dtype, _requires_grad, _shape = attrgetter("dtype"), attrgetter("requires_grad"), attrgetter("shape")
_contiguous, _index, _numel, _pointer = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.numel, torch.Tensor.data_ptr


def _scales_at(rows, cols):
    return (_HEAD + rows * (-(-cols // 32) * 16) + 127) // 128 * 128


def _packed_bytes(format, rows, cols):
    return _scales_at(rows, cols) + -(-rows // 128) * -(-cols // (4 * _BLOCK[format])) * 512


class Fp4Matrix:
    """A matrix in 4 bits on the GPU: `data` (uint8, contiguous) holds the packed form that include/bitsqz_llm_c.h describes, of `rows` x `cols`
    elements in `format` (MXFP4 or NVFP4).  The tensor may be saved, sent and loaded as it is."""

    __slots__ = ("data", "rows", "cols", "format")

    def __init__(self, data, rows, cols, format=NVFP4):
        if format not in _BLOCK:
            raise ValueError("format must be MXFP4 (8) or NVFP4 (9)")
        if rows < 0 or cols < 1 or rows > 0x7fffff00 or cols > 0x7fffff00:
            raise ValueError("a matrix has 0 to 2^31 - 256 rows and 1 to 2^31 - 256 columns")
        if data.dtype != torch.uint8 or not data.is_cuda or not data.is_contiguous() or data.numel() < _packed_bytes(format, rows, cols) or data.data_ptr() % 16:
            raise ValueError("data must be a contiguous uint8 CUDA tensor of at least %d bytes on a 16-byte boundary" % _packed_bytes(format, rows, cols))
        self.data, self.rows, self.cols, self.format = data, rows, cols, format

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def nbytes(self):
        return _packed_bytes(self.format, self.rows, self.cols)

    @property
    def tensor_scale(self):
        """The matrix scale (a float32 view of one element)."""
        return self.data[:4].view(torch.float32)

    @property
    def codes(self):
        """The codes, two to a byte (a view, rows x 16 bytes for 32 columns)."""
        ld = -(-self.cols // 32) * 16
        return self.data[_HEAD: _HEAD + self.rows * ld].view(self.rows, ld)

    def block_scales(self):
        """The scale bytes in the order of the blocks (a copy, rows x blocks)."""
        blocks = -(-self.cols // _BLOCK[self.format])
        groups, quads, at = -(-self.rows // 128), -(-blocks // 4), _scales_at(self.rows, self.cols)
        tiles = self.data[at: at + groups * quads * 512].view(groups, quads, 32, 4, 4)
        return tiles.permute(0, 3, 2, 1, 4).reshape(groups * 128, quads * 4)[: self.rows, :blocks].contiguous()


_entries = {}                                             # C entries by name, looked up once


def _entry(name):
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(lib(), name)
    return f


def _call(name, index, *args):
    """A C entry on the current stream of device `index` (its last argument), with that device current."""
    f = _entries.get(name) or _entry(name)
    if _device() == index:
        rc = f(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _stream(index))
    if rc != 0:
        raise RuntimeError(name + " failed")


def _rows(x, what):
    """(rows, cols, row stride) of a tensor whose leading dimensions lie as the rows of one matrix."""
    if not x.is_cuda or x.dtype not in _TYPES:
        raise ValueError("%s must be a float32, float16 or bfloat16 CUDA tensor" % what)
    dim = x.dim()
    if dim == 0 or x.size(-1) == 0:
        raise ValueError("%s must have at least one dimension and one column" % what)
    if dim > 2:
        try:
            x = x.view(x.numel() // x.size(-1), x.size(-1))
        except RuntimeError:
            raise ValueError("the leading dimensions of %s do not lie as the rows of one matrix: pass a contiguous tensor" % what) from None
    elif dim == 1:
        x = x.view(1, -1)
    rows, cols = x.shape
    ld, inner = x.stride()
    if cols > 1 and inner != 1 or rows > 1 and ld < cols:
        raise ValueError("rows of %s must be contiguous and must not overlap" % what)
    return rows, cols, ld


def _span(t):
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else t.data_ptr()


def _result(out, shape, dtype, device, *inputs):
    """The tensor that a call writes, and its row stride: a new one, or the caller's after a look at it."""
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    if out is None:
        return inputs[0].new_empty(shape, dtype=dtype), shape[-1]
    if out.dtype != dtype or tuple(out.shape) != tuple(shape) or out.device != device or out.requires_grad:
        raise ValueError("out must be a %s tensor of shape %s on %s that needs no gradient" % (dtype, tuple(shape), device))
    ld = shape[-1]
    if out.numel():
        ld = _rows(out, "out")[2]
        a, b = _span(out)
        for t in inputs:
            c, d = _span(t)
            if a < d and c < b:
                raise ValueError("out must not overlap an input")
        torch.autograd.graph.increment_version(out)
    return out, ld


def _packed(m, what):
    if not isinstance(m, Fp4Matrix):
        raise ValueError("%s must be an Fp4Matrix" % what)
    return m


def fp4_quantize(x, format=NVFP4, amax=None, out=None):
    """`x` (float32, float16 or bfloat16; the last dimension contiguous, leading dimensions are rows) in 4 bits, as an Fp4Matrix.

    MXFP4: blocks of 32 along a row with power-of-two scales.  NVFP4: blocks of 16 with E4M3 scales, and a power-of-two scale for the matrix
    that comes from its largest magnitude: found in a pass in front, or given as `amax` (a float32 CUDA tensor of one element, from
    calibration; larger elements saturate).  Elements go to the nearest code, ties to even.  A block with Inf or NaN reads back as NaN.
    `out`: an Fp4Matrix of the same shape and format to write."""
    if format not in _BLOCK:
        raise ValueError("format must be MXFP4 (8) or NVFP4 (9)")
    rows, cols, ld = _rows(x, "x")
    device = x.device
    if amax is not None and (format != NVFP4 or amax.dtype != torch.float32 or amax.numel() != 1 or amax.device != device):
        raise ValueError("amax is a float32 tensor of one element on x's device, for NVFP4")
    if out is None:
        out = Fp4Matrix.__new__(Fp4Matrix)
        out.data, out.rows, out.cols, out.format = x.new_empty(_packed_bytes(format, rows, cols), dtype=torch.uint8), rows, cols, format
    else:
        if _packed(out, "out").shape != (rows, cols) or out.format != format or out.data.device != device:
            raise ValueError("out must be an Fp4Matrix of %d x %d in the same format on x's device" % (rows, cols))
        a, b = _span(out.data)
        for t in (x,) if amax is None else (x, amax):
            c, d = _span(t)
            if a < d and c < b:
                raise ValueError("out must not overlap an input")
        torch.autograd.graph.increment_version(out.data)
    type = _TYPES[x.dtype]
    need = _entry("bsq_fp4_scratch_bytes")(format, type, rows, cols) if amax is None and format == NVFP4 else 0
    scratch = x.new_empty(need, dtype=torch.uint8) if need else None
    _call("bsq_fp4_quantize", device.index, format, x.data_ptr(), type, rows, cols, ld, None if amax is None else amax.data_ptr(), out.data.data_ptr(),
          None if scratch is None else scratch.data_ptr())
    return out


def fp4_dequantize(m, dtype=torch.float32, out=None):
    """The values of an Fp4Matrix: (element * block scale) * matrix scale in FP32, rounded once to `dtype`."""
    _packed(m, "m")
    device = m.data.device
    out, ld = _result(out, (m.rows, m.cols), dtype, device, m.data)
    _call("bsq_fp4_dequantize", device.index, m.format, m.data.data_ptr(), m.rows, m.cols, out.data_ptr(), _TYPES[dtype], ld)
    return out


def fp4_matmul(a, b, dtype=torch.bfloat16, out=None):
    """a b^T of two Fp4Matrix of one format with the same number of columns: (a.rows, b.rows) in `dtype`, summed in FP32 and rounded once
    (float32 results of more than 4096 columns: at every 4096, added up in FP32)."""
    _packed(a, "a")
    _packed(b, "b")
    device = a.data.device
    if a.format != b.format or a.cols != b.cols or b.data.device != device:
        raise ValueError("a and b must have the same format, number of columns and device")
    out, ld = _result(out, (a.rows, b.rows), dtype, device, a.data, b.data)
    _call("bsq_fp4_matmul", device.index, a.format, a.data.data_ptr(), a.rows, b.data.data_ptr(), b.rows, a.cols, out.data_ptr(), _TYPES[dtype], ld, None)
    return out


def _grad(name, dy, m, packed_rows, out_rows, dtype, out):
    _packed(m, "the packed operand")
    if dy.dtype != torch.bfloat16 or not dy.is_cuda or dy.device != m.data.device:
        raise ValueError("dy must be a bfloat16 tensor on the packed operand's device")
    if dy.dim() == 0 or dy.size(-1) == 0:
        raise ValueError("dy must have at least one dimension and one column")
    if dy.numel():
        M, N, ld = _rows(dy, "dy")
    else:
        M, N, ld = 0, dy.size(-1), dy.size(-1)
    if packed_rows(M, N) != m.rows:
        raise ValueError("dy is %d x %d and the packed operand %d x %d" % (M, N, m.rows, m.cols))
    device = dy.device
    shape = tuple(dy.shape[:-1]) + (m.cols,) if out_rows is None else (out_rows(M, N), m.cols)
    out, ld_out = _result(out, shape, dtype, device, dy, m.data)
    p = dy.data_ptr()
    need = _entry("bsq_fp4_grad_scratch_bytes")(p, M, N, ld) if M and (p % 16 or ld % 8) else 0
    scratch = m.data.new_empty(need) if need else None
    s = None if scratch is None else scratch.data_ptr()
    if out_rows is None:
        _call(name, device.index, m.format, p, M, ld, m.data.data_ptr(), N, m.cols, out.data_ptr(), _TYPES[dtype], ld_out, s, None)
    else:
        _call(name, device.index, m.format, p, M, N, ld, m.data.data_ptr(), m.cols, out.data_ptr(), _TYPES[dtype], ld_out, s, None)
    return out


def fp4_grad_input(dy, w, dtype=torch.bfloat16, out=None):
    """dy w: the gradient of the input of y = x w^T from dy (bfloat16, (..., w.rows)) and the packed weight, (..., w.cols) in `dtype`.  The weight's
    values are exact in bfloat16; sums are FP32, rounded once (float32 results: at every 1024 terms, added up in FP32)."""
    return _grad("bsq_fp4_grad_input", dy, w, lambda M, N: N, None, dtype, out)


def fp4_grad_weight(dy, x, dtype=torch.bfloat16, out=None):
    """dy^T x: the gradient of the weight from dy (bfloat16, (..., N) with x.rows rows in all) and the packed activations, (N, x.cols) in `dtype`,
    summed as in fp4_grad_input."""
    return _grad("bsq_fp4_grad_weight", dy, x, lambda M, N: M, lambda M, N: N, dtype, out)


def _laid_out(x):
    """x, or a copy where its elements do not lie as the rows of one matrix (a transposed or broadcast tensor)."""
    if not x.is_contiguous():
        try:
            _rows(x, "x")
        except ValueError:
            return x.contiguous()
    return x


class _Fp4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, w4, format):
        x4 = fp4_quantize(x, format)
        if w4 is None:
            w4 = fp4_quantize(weight, format)
        ctx.x_shape, ctx.sizes, ctx.format, ctx.dtype = x.shape, (x4.rows, w4.rows, w4.cols), format, None if weight is None else weight.dtype
        # parked until the backward pass: 4 bits an element instead of 16
        ctx.save_for_backward(x4.data if ctx.needs_input_grad[1] else None, w4.data if ctx.needs_input_grad[0] else None)
        return fp4_matmul(x4, w4, x.dtype).view(x.shape[:-1] + (w4.rows,))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x_data, w_data = ctx.saved_tensors
        M, N, K = ctx.sizes
        dy = dy.reshape(M, N)                                # (a copy where dy is broadcast, as the gradient of a sum is)
        if not dy.is_contiguous():
            dy = dy.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = fp4_grad_input(dy, Fp4Matrix(w_data, N, K, ctx.format)).view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dw = fp4_grad_weight(dy, Fp4Matrix(x_data, M, K, ctx.format), ctx.dtype)
        return dx, dw, None, None


def fp4_linear(x, weight, format=NVFP4):
    """x w^T with both operands in 4 bits, under autograd: x (bfloat16, (..., K)), weight either a tensor (N, K) that is quantised in every call and
    gets a gradient of its own type, or an Fp4Matrix that is frozen.  The backward pass treats quantisation as the identity: dx = dy q(w), dw = dy^T q(x),
    where q(x) is kept in 4 bits between the passes.  x or a weight whose elements do not lie as the rows of one matrix is copied first.  Autocast does not change what
    is asked of x: pass it in bfloat16."""
    if x.dtype != torch.bfloat16 or not x.is_cuda:
        raise ValueError("x must be a bfloat16 CUDA tensor")
    if isinstance(weight, Fp4Matrix):
        if weight.format != format or x.dim() == 0 or x.size(-1) != weight.cols:
            raise ValueError("the weight must be packed in `format` with as many columns as x")
        return _Fp4Linear.apply(_laid_out(x), None, weight, format)
    if weight.dim() != 2 or x.dim() == 0 or x.size(-1) != weight.size(1) or weight.device != x.device or not weight.size(0):
        raise ValueError("the weight must be a (N, K) tensor on x's device, K the last dimension of x")
    return _Fp4Linear.apply(_laid_out(x), _laid_out(weight), None, format)


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_XENT_COLS, _XENT_TOKENS = 65536, {torch.float16: 65536, torch.bfloat16: 524288}


def _scratch(name, device, *args):
    """The scratch that an entry wants for `args`."""
    f = _entries.get(name) or _entry(name)
    if _device() == device.index:
        need = f(*args)
    else:
        with torch.cuda.device(device):
            need = f(*args)
    return torch.empty(need, dtype=torch.uint8, device=device)


def _xent_operands(x, weight):
    rows, cols, ld = _rows(x, "x") if x.numel() else (0, x.size(-1), x.size(-1))
    vocab, _, ld_w = _rows(weight, "weight")
    return _TYPES[x.dtype], x.data_ptr(), rows, cols, ld, weight.data_ptr(), vocab, ld_w


def _xent_loss(x, weight, target, ignore_index, label_smoothing, reduction):
    """The loss, and what the gradient wants beside it."""
    device, operands = x.device, _xent_operands(x, weight)
    loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=device)
    stats = torch.empty(2 * operands[2] + 1, dtype=torch.float32, device=device)
    scratch = _scratch("bsq_linear_xent_scratch_bytes", device, *operands, label_smoothing)
    _call("bsq_linear_xent", device.index, *operands, target.data_ptr(), ignore_index, label_smoothing, reduction, loss.data_ptr(), stats.data_ptr(), scratch.data_ptr(), None)
    return loss, stats


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, label_smoothing, reduction):
        loss, stats = _xent_loss(x, weight, target, ignore_index, label_smoothing, reduction)
        ctx.save_for_backward(x, weight, target, stats)
        ctx.how = ignore_index, label_smoothing, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, target, stats = ctx.saved_tensors
        device, (want_x, want_w) = x.device, ctx.needs_input_grad[:2]
        x, weight = _laid_out(x) if x.numel() else x, _laid_out(weight)      # (hooks may bring back other tensors than were saved)
        operands, grad, cols = _xent_operands(x, weight), grad.contiguous(), x.size(-1)          # (grad: one value for all tokens where the losses were added up)
        dx = x.new_empty(x.shape) if want_x else None
        dw = weight.new_empty(weight.shape) if want_w else None
        scratch = _scratch("bsq_linear_xent_grad_scratch_bytes", device, *operands, 1 if want_x else 0)
        _call("bsq_linear_xent_grad", device.index, *operands, target.data_ptr(), *ctx.how, stats.data_ptr(), grad.data_ptr(), None if dx is None else dx.data_ptr(), cols,
              None if dw is None else dw.data_ptr(), cols, scratch.data_ptr(), None)
        return dx, dw, None, None, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """Softmax cross entropy of the logits x weight^T without keeping them, under autograd: x (float16 or bfloat16, (..., D)), weight (V, D) of the same type, target int64
    of x's leading dimensions.  A token's loss is lse - (1 - e) * logit of its target - e * mean of its logits, e = label_smoothing, in float32; tokens whose target is
    ignore_index have 0.  reduction "none": each token's (the log probability of a given token is its negative), "sum", or "mean" over the tokens that are not ignored (none of them:
    NaN).  A target outside 0 .. V - 1 gives NaN for its token.  Logits are FP32 sums; the backward pass computes them again, rounds their gradient to the type of x and returns the gradients of x and
    weight in it, rounded once.  Hidden states of ignored tokens get a gradient of 0; they are multiplied by 0 on the way to the weight's and have to be finite.
    At most 65536 columns and 65536 (float16) or 524288 (bfloat16) tokens.  Tensors that do not lie as the rows of one matrix are copied first.  Autocast does not change what is
    asked of x: pass it and the weight in 16 bits.  Forward-mode derivatives are refused (NotImplementedError)."""
    if x.dtype not in _XENT_TOKENS or not x.is_cuda or x.dim() == 0 or x.size(-1) == 0:
        raise ValueError("x must be a float16 or bfloat16 CUDA tensor with at least one column")
    if weight.dim() != 2 or weight.dtype != x.dtype or weight.device != x.device or weight.size(1) != x.size(-1) or not weight.size(0):
        raise ValueError("the weight must be a (V, D) tensor of x's type on x's device, D the last dimension of x")
    if target.dtype != torch.int64 or target.device != x.device or target.shape != x.shape[:-1]:
        raise ValueError("target must be an int64 tensor of x's leading dimensions on x's device")
    if reduction not in _REDUCTIONS:
        raise ValueError('reduction must be "none", "sum" or "mean"')
    label_smoothing, ignore_index = float(label_smoothing), int(ignore_index)
    if not 0.0 <= label_smoothing <= 1.0 or not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError("label_smoothing must be within 0 and 1, ignore_index an int64")
    if x.size(-1) > _XENT_COLS or target.numel() > _XENT_TOKENS[x.dtype]:
        raise ValueError("at most %d columns and %d tokens: split the batch" % (_XENT_COLS, _XENT_TOKENS[x.dtype]))
    call = _laid_out(x) if x.numel() else x, _laid_out(weight), target.contiguous(), ignore_index, label_smoothing, _REDUCTIONS[reduction]
    # (a tensor with a forward-mode tangent need not require a gradient: the function refuses it)
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled() or unpack_dual(x).tangent is not None or unpack_dual(weight).tangent is not None:
        return _LinearCrossEntropy.apply(*call)
    return _xent_loss(*call)[0]


def _dense(t):
    """Whether a tensor's elements fill one run of memory, in whatever order."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _overlap(grads, to):
    """Why the library refused a list: whether a tensor that is written shares memory with another one."""
    spans = [(*_span(o), True) for o in to] + [(*_span(g), False) for g, o in zip(grads, to) if g.data_ptr() != o.data_ptr()]
    spans = sorted(s for s in spans if s[0] < s[1])
    any_end = out_end = 0
    for a, b, written in spans:
        if a < (any_end if written else out_end):
            return True
        any_end, out_end = max(any_end, b), max(out_end, b if written else 0)
    return False


def clip_grad_norm(grads, max_norm, norm_type=2.0, out=None):
    """The norm of `grads` (float32, float16 or bfloat16 CUDA tensors of one device, mixed as they come) taken as one vector, as a float32 tensor of no
    dimensions; the gradients are multiplied by min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out` (of the same types;
    contiguous with as many elements, or of the same shapes and strides).  norm_type 2 or math.inf.  max_norm None: the norm alone.
    What is scaled in place must not need a gradient itself: these are the parameters' gradients, not the parameters.
    As with torch.nn.utils.clip_grad_norm_ a NaN in any gradient makes the norm and all gradients NaN; an Inf makes the norm Inf, the finite gradients 0 and only the
    infinite elements NaN.  To skip a step that went wrong look at the norm, not at a gradient."""
    grads = list(grads)
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError("norm_type must be 2 or infinity")
    if not grads:
        raise ValueError("no gradients: the device of their norm is not known")
    if max_norm is None and out is not None:
        raise ValueError("out needs a max_norm")
    max_norm = None if max_norm is None else float(max_norm)
    if max_norm is not None and not max_norm >= 0:
        raise ValueError("max_norm must not be negative or NaN")
    device, n = grads[0].device, len(grads)
    # (an attribute of all of them at a time: a few hundred gradients are looked at in every step)
    index, dtypes, plain = grads[0].get_device(), list(map(_dtype, grads)), list(map(_contiguous, grads))
    types = [_TYPES.get(d, -1) for d in dtypes]
    if index < 0 or min(types) < 0 or set(map(_index, grads)) != {index} or not (all(plain) or all(p or _dense(g) for p, g in zip(plain, grads))):
        raise ValueError("gradients must be dense float32, float16 or bfloat16 CUDA tensors on one device")
    if max_norm is not None and out is None and any(map(_requires_grad, grads)):
        raise ValueError("tensors that are scaled in place must need no gradient (pass the parameters' gradients, not the parameters; detached ones if they need gradients themselves)")
    counts, ptrs = array("Q", map(_numel, grads)), array("Q", map(_pointer, grads))
    to, outs = grads, ptrs
    if out is not None:
        to = list(out)
        if len(to) != n:
            raise ValueError("out must have a tensor for each gradient")
        if list(map(_dtype, to)) != dtypes or set(map(_index, to)) != {index} or any(map(_requires_grad, to)):
            raise ValueError("tensors of out must have the type and device of their gradients, and need no gradient")
        if not (all(plain) and all(map(_contiguous, to))) and [(o.shape, o.stride()) for o in to] != [(g.shape, g.stride()) for g in grads]:
            raise ValueError("tensors of out that are not contiguous must have the shape and strides of their gradients")
        if array("Q", map(_numel, to)) != counts:
            raise ValueError("tensors of out must have as many elements as their gradients")
        outs = array("Q", map(_pointer, to))
    types = array("i", types)
    norm = torch.empty((), dtype=torch.float32, device=device)
    scratch = torch.empty(_NORM_SCRATCH, dtype=torch.uint8, device=device)
    try:
        _call("bsq_grad_norm_clip", index, ptrs.buffer_info()[0], counts.buffer_info()[0], types.buffer_info()[0], n, None if max_norm is None else outs.buffer_info()[0],
              0.0 if max_norm is None else max_norm, 0 if norm_type == math.inf else 2, norm.data_ptr(), scratch.data_ptr())
    except RuntimeError:
        if max_norm is not None and _overlap(grads, to):
            raise ValueError("the tensors that are written must not overlap one another or another gradient") from None
        raise
    if max_norm is not None:
        torch.autograd.graph.increment_version(to)
    return norm


_QUINTIC = (3.4445, -4.7750, 2.0315)
_ORTH_SIDE, _ORTH_STEPS = 65536, 64


def orthogonalize(updates, steps=5, coefficients=_QUINTIC, eps=1e-7, scale=1.0, dtype=torch.bfloat16, out=None):
    """Updates with their singular values brought near 1 by Newton-Schulz steps: X = G / (|G| + eps), then `steps` times X <- a X + (b A + c A^2) X with A = X X^T (from the
    right with X^T X where G has more rows than columns), times `scale`.  `updates`: a tensor of at least two dimensions (the leading ones are a stack of matrices) or a list of them
    (float32, float16 or bfloat16 CUDA tensors of one device, of any shapes); the result is of the same form, in `dtype`.  Matrices of one shape and type go through together.  coefficients: (a, b, c)
    for all steps, or one triple for each; they must keep singular values from 0 to 1 below 1000.  `out`: tensors to write, apart from each other and from the updates (side by side in the rows of one tensor they may lie; without it,
    results of one shape that follow one another in a list lie in one allocation, which is freed with the last of them).

    bfloat16 results are off by at most about half their own rounding beside it: X is held in 2 x 16 bits, products read 16 and sum in FP32 (a side of up to 128: products of 22 bits); of exactly
    rank one up to 3.5e-3 in all, with both sides above 128 up to 1.2e-2 where those of a row or column take few values, whose roundings do not average out.
    float32 and float16 results come from products of 2 x 16 bits of every operand, three times the work (1e-6 to 2e-4 off, more the further singular values lie apart; up to 1.2e-3 for rank one of few values).  An Inf or NaN makes its whole matrix NaN; zeros stay zeros, and where |G| is far below eps the result may be 0.
    Matrices whose rows are not contiguous are copied first.  The result needs no gradient and gives none to the updates, backwards or forwards.  Sides of at most 65536, 1 to 64 steps."""
    single = isinstance(updates, torch.Tensor)
    updates = [updates] if single else list(updates)
    if not 1 <= steps <= _ORTH_STEPS or int(steps) != steps:
        raise ValueError("steps must be a whole number from 1 to 64")
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    table = list(coefficients)
    table = [table] * int(steps) if len(table) == 3 and all(isinstance(v, (int, float)) for v in table) else table
    if len(table) != steps or any(isinstance(t, (int, float)) or len(t) != 3 for t in table):
        raise ValueError("coefficients must be (a, b, c), or one such triple for each step")
    eps, scale = float(eps), float(scale)
    if not 0.0 <= eps < math.inf or not math.isfinite(scale):
        raise ValueError("eps must be finite and not negative, scale finite")
    if not updates:
        return []
    # (an attribute of all of them at a time: a step has a few hundred matrices)
    device, index, n = updates[0].device, updates[0].get_device(), len(updates)
    dtypes, shapes = list(map(_dtype, updates)), list(map(_shape, updates))
    if index < 0 or set(map(_index, updates)) != {index} or not _TYPES.keys() >= set(dtypes) or any(len(s) < 2 or s[-1] > _ORTH_SIDE or s[-2] > _ORTH_SIDE for s in shapes):
        raise ValueError("updates must be float32, float16 or bfloat16 CUDA tensors on one device of at least two dimensions, with sides of at most 65536")
    if out is None:
        outs, at = [], 0
        while at < n:                                            # (neighbours of one shape from one allocation: a call of the allocator costs more than a matrix's other arguments)
            shape, end = shapes[at], at + 1
            while end < n and shapes[end] == shape and shape[0]:
                end += 1
            some = torch.empty((shape[0] * (end - at),) + shape[1:], dtype=dtype, device=device)
            outs += [some] if end == at + 1 else some.unsafe_split(shape[0])                      # (tensors of their own, not views of one that count their changes together)
            at = end
    else:
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(outs) != n or isinstance(out, torch.Tensor) != single:
            raise ValueError("out must have the form of updates")
        if set(map(_dtype, outs)) != {dtype} or list(map(_shape, outs)) != shapes or set(map(_index, outs)) != {index} or any(map(_requires_grad, outs)):
            raise ValueError("tensors of out must have the shapes of the updates, dtype %s, their device, and need no gradient" % dtype)
    keep = updates                                               # (until the call has been enqueued)
    if all(map(_contiguous, updates)) and all(map(_contiguous, outs)) and all(len(s) == 2 and s[0] and s[1] for s in shapes):
        ins, tos = array("Q", map(_pointer, updates)), array("Q", map(_pointer, outs))
        rows, cols, types = array("Q", [s[0] for s in shapes]), array("Q", [s[1] for s in shapes]), array("i", [_TYPES[d] for d in dtypes])
        lds = ld_outs = cols
    else:
        ins, rows, cols, lds, types, tos, ld_outs, keep = array("Q"), array("Q"), array("Q"), array("Q"), array("i"), array("Q"), array("Q"), []
        for g, o in zip(updates, outs):
            if not g.numel():
                continue
            if not _stacked(g):
                g = g.contiguous()
                keep.append(g)
            if not _stacked(o):
                raise ValueError("rows of out must be contiguous and must not overlap")
            m, k, size, to_size = g.size(-2), g.size(-1), g.element_size(), o.element_size()
            for a, b in zip(_matrices(g), _matrices(o)):
                ins.append(g.data_ptr() + a * size)
                tos.append(o.data_ptr() + b * to_size)
            count = g.numel() // (m * k)
            rows.extend([m] * count), cols.extend([k] * count), types.extend([_TYPES[g.dtype]] * count)
            lds.extend([g.stride(-2) if m > 1 else k] * count), ld_outs.extend([o.stride(-2) if m > 1 else k] * count)
    if ins:
        flat = array("f", [v for t in table for v in t])
        arrays = [a.buffer_info()[0] for a in (ins, rows, cols, lds, types, tos, ld_outs, flat)]
        scratch = _scratch("bsq_orthogonalize_scratch_bytes", device, arrays[1], arrays[2], arrays[4], len(ins), _TYPES[dtype])
        call = (*arrays[:5], len(ins), *arrays[5:7], _TYPES[dtype], int(steps), arrays[7], eps, scale)
        try:
            _call("bsq_orthogonalize", index, *call, scratch.data_ptr(), None)
        except RuntimeError:
            why = lib().bsq_orthogonalize_check(*call)
            if why == 2:
                raise ValueError("coefficients must keep singular values from 0 to 1 below 1000") from None
            if why == 3:
                raise ValueError("the matrices that are written must lie apart from one another and from the updates") from None
            raise
    if out is not None:
        torch.autograd.graph.increment_version(outs)
    return outs[0] if single else outs


def _stacked(t):
    """Whether every matrix of a stack has contiguous rows that do not overlap."""
    return (t.stride(-1) == 1 or t.size(-1) == 1) and (t.size(-2) == 1 or t.stride(-2) >= t.size(-1))


def _matrices(t):
    """Where the matrices of a stack begin, in elements from its first."""
    at = [0]
    for n, s in zip(t.shape[:-2], t.stride()[:-2]):
        at = [a + i * s for a in at for i in range(n)]
    return at
