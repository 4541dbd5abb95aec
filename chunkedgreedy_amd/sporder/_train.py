"""Operators of a training step around the SpMM: row lookup, layer norm and
the orthogonalisation of a weight's update, each with what its backward pass
needs.  They have no counterpart in the reference.

Unlike the rest of the package they run on torch's current stream of the
input's device and return without waiting, so they follow and precede torch
operations on that stream and can be captured into a graph.  Outputs and
scratch come from torch's allocator.  They take no Context.  Inputs are torch
GPU tensors, or DLPack-capable GPU arrays.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._sporder import _as_tensor

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16,
          torch.float16: _lib.TYPE_F16}
_TOKEN_BITS = {torch.int32: 32, torch.int64: 64}


class _BadArgument(ValueError):
    pass


def _floats(a, name):
    t = _as_tensor(a, name)
    if not t.is_cuda:
        raise TypeError(f"{name} must be a GPU tensor")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return t


def _token_ids(a, ref):
    t = _as_tensor(a, "tokens")
    if not t.is_cuda:
        raise TypeError("tokens must be a GPU tensor")
    if t.dtype not in _TOKEN_BITS:
        raise TypeError(f"tokens must be int32 or int64, got {t.dtype}")
    _same_device(t, ref, "tokens")
    return t if t.is_contiguous() else t.contiguous()


def _same_device(t, ref, name):
    if t.device != ref.device:
        raise ValueError(f"{name} lives on {t.device}, expected {ref.device}")


def _rows(t):
    """(tensor, rows, stride): `t` as rows of its last dimension a fixed number
    of elements apart, copied only where its strides allow no such view."""
    dim = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // dim, dim
    if t.dim() == 2 and (t.stride(1) == 1 or dim == 1):
        return t, t.shape[0], t.stride(0)
    t = t.contiguous()
    return t, t.numel() // dim, dim


def _out(out, shape, dtype, ref):
    if out is None:
        if shape == ref.shape and dtype == ref.dtype and ref.is_contiguous():
            return torch.empty_like(ref)  # half the time of an allocation from parts
        return ref.new_empty(shape, dtype=dtype)
    if (not isinstance(out, torch.Tensor) or out.shape != torch.Size(shape) or out.dtype != dtype
            or out.device != ref.device or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                         f"{ref.device}")
    return out


# The current stream's handle without a Stream object around it (a call less
# than a microsecond long instead of a few).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


_entries = {}


def _call(name, ref, *args):
    """Queues a C entry on the current stream of ref's device."""
    index = ref.get_device()
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        rc = fn(_raw_stream(index), *args)
    else:
        with torch.cuda.device(index):
            rc = fn(_raw_stream(index), *args)
    if rc == _lib.BAD_ARGUMENT:
        raise _BadArgument(f"{name} refused its arguments")
    if rc != _lib.OK:
        raise RuntimeError(f"{name} returned {rc}")


def embedding(table, tokens, *, scale=1.0, out=None):
    """Rows of a table by token: out[..., :] = scale * table[tokens[...]].

    Arguments:
        table: (rows, dim) float32, bfloat16 or float16; unit stride along dim
        tokens: int32 or int64 ids of any shape
        scale: factor applied in 32 bits before the one rounding to the type
        out: contiguous tensor of shape tokens.shape + (dim,), or None

    A token outside [0, rows) gives a row of NaN.  Returns out.
    """
    table = _floats(table, "table")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("table must be a (rows, dim) tensor of at least one element")
    tokens = _token_ids(tokens, table)
    rows, dim = table.shape
    out = _out(out, (*tokens.shape, dim), table.dtype, table)
    table, _, stride = _rows(table)
    _call("sporder_embedding", table, _TYPES[table.dtype], rows, dim, stride, table.data_ptr(),
          tokens.numel(), _TOKEN_BITS[tokens.dtype], tokens.data_ptr(), float(scale), dim,
          out.data_ptr())
    return out


def _padding_row(padding_idx, num_rows):
    if padding_idx is not None and not 0 <= padding_idx < num_rows:
        raise ValueError("padding_idx must be a row of the table")


def embedding_grad(grad, tokens, num_rows, *, scale=1.0, padding_idx=None, dtype=None, out=None):
    """Gradient of :func:`embedding` by its table, dense:
    out[v] = scale * sum of grad[t] over the tokens equal to v.

    Arguments:
        grad: tokens.shape + (dim,), float32, bfloat16 or float16
        tokens: int32 or int64 ids, at most 2^28 - 4096 of them; ids outside
            [0, num_rows) are left out
        num_rows: rows of the table
        padding_idx: a row in [0, num_rows) that gets no gradient, or None
        dtype: grad's type (default) or float32, the type of the result
        out: contiguous (num_rows, dim) tensor of that type, or None

    The sums are held in 32 bits.  Their order depends on the tokens, the sizes
    and grad's type, strides and alignment: the same call gives the same bits
    from run to run, the same values laid out otherwise may differ in the last
    ones.  Every row is written.  Returns out.
    """
    grad = _floats(grad, "grad")
    tokens = _token_ids(tokens, grad)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape or grad.shape[-1] < 1:
        raise ValueError("grad must have the tokens' shape and one more dimension")
    num_rows = int(num_rows)
    if not 1 <= num_rows <= 2**31 - 2:
        raise ValueError("num_rows must be in [1, 2^31 - 2]")
    _padding_row(padding_idx, num_rows)
    if dtype is None:
        dtype = grad.dtype
    elif dtype not in (grad.dtype, torch.float32):
        raise ValueError("dtype must be grad's type or float32")
    dim = grad.shape[-1]
    count = tokens.numel()
    out = _out(out, (num_rows, dim), dtype, grad)
    grad, _, stride = _rows(grad)
    size = _lib.load().sporder_embedding_grad_work_bytes(count, num_rows, dim)
    work = grad.new_empty(size, dtype=torch.uint8) if size else None
    _call("sporder_embedding_grad", grad, _TYPES[grad.dtype], count, dim, stride, grad.data_ptr(),
          _TOKEN_BITS[tokens.dtype], tokens.data_ptr(), float(scale),
          -1 if padding_idx is None else int(padding_idx), num_rows, _TYPES[dtype], dim,
          out.data_ptr(), work.data_ptr() if size else 0, size)
    return out


def _norm_vector(a, name, dim, ref):
    t = _floats(a, name)
    if t.dtype not in (ref.dtype, torch.float32):
        raise TypeError(f"{name} must have x's type or float32, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != dim:
        raise ValueError(f"{name} must have shape ({dim},)")
    _same_device(t, ref, name)
    return t if t.is_contiguous() else t.contiguous()


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None):
    """Layer norm over the last dimension:
    y = (x - mean) * rstd * weight + bias, rstd = (var + eps)^-1/2.

    Arguments:
        x: (..., dim) float32, bfloat16 or float16; rows a fixed number of
            elements apart are read in place, other strides are copied
        weight, bias: (dim,) of x's type or float32 (both of one type), or None
        eps: >= 0
        out: contiguous tensor of x's shape and type, or None; may be x

    Returns (y, mean, rstd); mean and rstd are float32 of shape x.shape[:-1],
    as :func:`layer_norm_grad` takes them.
    Sums and squares are held in 32 bits: a row whose deviations from its mean
    pass some 1e19 has an infinite variance, and y is its bias.
    """
    x = _floats(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0")
    dim = x.shape[-1]
    if weight is not None:
        weight = _norm_vector(weight, "weight", dim, x)
    if bias is not None:
        bias = _norm_vector(bias, "bias", dim, x)
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError("weight and bias must have the same type")
    y = _out(out, x.shape, x.dtype, x)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    given = weight if weight is not None else bias
    x, rows, stride = _rows(x)
    _call("sporder_layer_norm", x, _TYPES[x.dtype],
          _lib.TYPE_F32 if given is None else _TYPES[given.dtype], rows, dim, stride,
          x.data_ptr(), 0 if weight is None else weight.data_ptr(),
          0 if bias is None else bias.data_ptr(), eps, dim, y.data_ptr(), mean.data_ptr(),
          rstd.data_ptr())
    return y, mean, rstd


def layer_norm_grad(grad, x, mean, rstd, weight=None):
    """Gradients of :func:`layer_norm`.

    Arguments:
        grad, x: the gradient by y and the forward call's x, of one shape and
            type
        mean, rstd: as the forward call returned them
        weight: as in the forward call

    Returns (dx, dweight, dbias): dx of x's type; dweight and dbias of
    weight's type (float32 without a weight), summed over all rows in 32 bits
    in an order that depends on the sizes and the inputs' types, strides and
    alignment: the same call gives the same bits from run to run.
    """
    x = _floats(x, "x")
    grad = _floats(grad, "grad")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    if grad.shape != x.shape:
        raise ValueError("grad must have x's shape")
    if grad.dtype != x.dtype:
        raise TypeError("grad must have x's type")
    _same_device(grad, x, "grad")
    dim = x.shape[-1]
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 \
                or t.shape != x.shape[:-1] or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name} must be the contiguous float32 tensor that layer_norm "
                             f"returned, of shape {tuple(x.shape[:-1])} on {x.device}")
    dtype = torch.float32
    if weight is not None:
        weight = _norm_vector(weight, "weight", dim, x)
        dtype = weight.dtype
    dx = _out(None, x.shape, x.dtype, x)
    dweight = x.new_empty(dim, dtype=dtype)
    dbias = torch.empty_like(dweight)
    x, rows, stride = _rows(x)
    grad, _, grad_stride = _rows(grad)
    size = _lib.load().sporder_layer_norm_grad_work_bytes(rows, dim)
    work = x.new_empty(size, dtype=torch.uint8)
    _call("sporder_layer_norm_grad", x, _TYPES[x.dtype], _TYPES[dtype], rows, dim, grad_stride,
          grad.data_ptr(), stride, x.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
          0 if weight is None else weight.data_ptr(), dim, dx.data_ptr(), dweight.data_ptr(),
          dbias.data_ptr(), work.data_ptr(), size)
    return dx, dweight, dbias


def _matrices(g, name):
    """`g` if newton_schulz takes it."""
    g = _floats(g, name)
    if g.dim() not in (2, 3) or g.shape[-1] < 1 or g.shape[-2] < 1 \
            or max(g.shape[-2:]) > 65536 or (g.dim() == 3 and g.shape[0] > 32768):
        raise ValueError(f"{name} must be (rows, cols) or (batch, rows, cols) with sides of 1 to "
                         "65536 and a batch of at most 32768")
    return g


def _step_count(steps):
    steps = int(steps)
    if not 1 <= steps < 2**31:
        raise ValueError("steps must be >= 1 and below 2^31")
    return steps


def newton_schulz(g, *, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, out=None):
    """Orthogonalise a matrix by Newton-Schulz products (the Muon optimiser's
    update): X = g / (|g| + eps) with the Frobenius norm, then ``steps`` times
    X <- a X + (b A + c A A) X with A = X X^T.

    Every singular value s of g / |g| becomes p(p(...p(s))) with p(s) = a s +
    b s^3 + c s^5; the default coefficients take most of [0, 1] close to 1 in
    five steps.  Matrices taller than wide are handled as their transposes.

    Arguments:
        g: (rows, cols), or a batch (batch, rows, cols), float32, bfloat16 or
            float16, sides of at most 65536; read in place where its last
            dimension has unit stride
        steps: >= 1
        coefficients: (a, b, c); refused where a singular value in [0, 1], or
            one of A or b A + c A A, could pass 31 within the steps
        eps: >= 0
        out: contiguous tensor of g's shape and type, or None; may be g

    X is held in 32 bits whatever the type.  Products have operands of 22 bits
    and 32-bit sums: a term is within 2^-21 of itself, and within some 2^-37 of
    the bounds on the norms of its row and column, so small rows, columns and
    matrices keep their own accuracy.  The result is about as close as 32-bit
    products give it, or up to some 8 times as far where those have single
    terms and round once (a diagonal matrix).  Returns out.
    """
    g = _matrices(g, "g")
    steps = _step_count(steps)
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0")
    a, b, c = (float(v) for v in coefficients)
    batch = g.shape[0] if g.dim() == 3 else 1
    rows, cols = g.shape[-2:]
    out = _out(out, g.shape, g.dtype, g)
    if g.stride(-1) != 1 and cols > 1:
        g = g.contiguous()
    lib = _lib.load()
    size = lib.sporder_newton_schulz_work_bytes(batch, rows, cols)
    work = g.new_empty(size, dtype=torch.uint8) if size else None
    try:
        _call("sporder_newton_schulz", g, _TYPES[g.dtype], batch, rows, cols,
              g.stride(0) if g.dim() == 3 else 0, g.stride(-2), g.data_ptr(), steps, a, b, c,
              float(eps), out.data_ptr(), work.data_ptr() if size else 0, size)
    except _BadArgument:
        raise ValueError(f"coefficients {(a, b, c)} take singular values past 31 within "
                         f"{steps} steps") from None
    return out
