"""Operators of a training step around the SpMM: row lookup, layer norm, the
orthogonalisation of a weight's update, dropout, the norms around a block and
the cross entropy of linear logits, each with what its backward pass needs.
They have no counterpart in the reference.

Unlike the rest of the package they run on torch's current stream of the
input's device and return without waiting, so they follow and precede torch
operations on that stream and can be captured into a graph.  Outputs and
scratch come from torch's allocator.  They take no Context.  Inputs are torch
GPU tensors, or DLPack-capable GPU arrays.
"""

from __future__ import annotations

import functools

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
    if t.get_device() != ref.get_device():  # of GPU tensors; a third of device's time
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
# The current device where a GPU tensor is at hand, so that torch is initialised.
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


_entries = {}


def _call(name, ref, *args):
    """Queues a C entry on the current stream of ref's device."""
    index = ref.get_device()
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if index == _device():
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


def _seed_words(seed, offset):
    """(seed, offset, state): host words, and a GPU tensor of two more or None."""
    offset = int(offset)
    if not 0 <= offset < 2**63:
        raise ValueError("offset must be in [0, 2^63)")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or not seed.is_cuda \
                or not seed.is_contiguous():
            raise ValueError("a seed on the GPU must be a contiguous int64 tensor (seed, offset)")
        return 0, offset, seed
    seed = int(seed)
    if not 0 <= seed < 2**64:
        raise ValueError("seed must be in [0, 2^64)")
    return seed, offset, None


def dropout(x, p, seed, *, offset=0, residual=None, out=None):
    """Dropout whose mask follows from a counter and is never stored:
    out = residual + (kept ? x / (1 - p) : 0).

    Arguments:
        x: float32, bfloat16 or float16 of any shape
        p: probability of being dropped, in [0, 1] (in steps of 2^-32)
        seed: int in [0, 2^64), or an int64 GPU tensor (seed, offset) that is
            read when the work runs, so that a captured graph's replays can
            each have another
        offset: int in [0, 2^63), added to the tensor's; calls that are to drop
            different elements under one seed have different offsets
        residual: tensor of x's shape and type, or None
        out: contiguous tensor of x's shape and type, or None; may be x or
            residual

    An element is kept by its index in x's shape alone (not by its type or
    strides), so the gradient by x is ``dropout(grad, p, seed, offset=offset)``.
    Dropped elements are 0 whatever x is there.  Returns out.
    """
    x = _floats(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1]")
    seed, offset, state = _seed_words(seed, offset)
    if state is not None:
        _same_device(state, x, "seed")
    if residual is not None:
        residual = _floats(residual, "residual")
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
        if residual.dtype != x.dtype:
            raise TypeError("residual must have x's type")
        _same_device(residual, x, "residual")
    out = _out(out, x.shape, x.dtype, x)
    if x.numel() == 0:
        return out
    if x.dim() == 0:
        x, residual = x[None], None if residual is None else residual[None]
    dim = x.shape[-1]
    x, rows, stride = _rows(x)
    residual_stride = 0
    if residual is not None:
        residual, _, residual_stride = _rows(residual)
    _call("sporder_dropout", x, _TYPES[x.dtype], rows, dim, stride, x.data_ptr(), residual_stride,
          0 if residual is None else residual.data_ptr(), p, seed, offset,
          0 if state is None else state.data_ptr(), dim, out.data_ptr())
    return out


def _block_inputs(x, gate, post_weight, weight, post_norm):
    """(gate, post_weight, weight, their type, whether the gate has rows)."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    dim = x.shape[-1]
    by_row = gate is not None and getattr(gate, "ndim", 1) == x.dim() > 1
    if by_row:
        gate = _like(gate, "gate", x)
    elif gate is not None:
        gate = _norm_vector(gate, "gate", dim, x)
    if post_weight is not None:
        if not post_norm:
            raise ValueError("post_weight is the weight of the norm that post_norm=False leaves out")
        post_weight = _norm_vector(post_weight, "post_weight", dim, x)
    if weight is not None:
        weight = _norm_vector(weight, "weight", dim, x)
    kind = None
    for t in (None if by_row else gate, post_weight, weight):
        if t is not None:
            if kind is not None and t.dtype != kind:
                raise TypeError("weights and a gate of shape (dim,) must have the same type")
            kind = t.dtype
    return gate, post_weight, weight, kind or torch.float32, by_row


def _like(a, name, x):
    t = _floats(a, name)
    if t.shape != x.shape:
        raise ValueError(f"{name} must have x's shape")
    if t.dtype != x.dtype:
        raise TypeError(f"{name} must have x's type")
    _same_device(t, x, name)
    return t


def _row_args(t):
    """(tensor to keep, stride, address) of an optional tensor of rows."""
    if t is None:
        return None, 0, 0
    t, _, stride = _rows(t)
    return t, stride, t.data_ptr()


def _address(t):
    return 0 if t is None else t.data_ptr()


def residual_norm(x, residual=None, gate=None, post_weight=None, weight=None, *, scale=1.0,
                  eps=1e-5, post_norm=True):
    """The norms after a block and before the next one, with the block's gate
    and residual scale:

        y = residual + scale * gate * post_weight * x * post_rstd
        h = weight * y * rstd

    with post_rstd = (mean x^2 + eps)^-1/2 and rstd = (mean y^2 + eps)^-1/2 of
    each row (root mean square norms).

    Arguments:
        x: (..., dim) float32, bfloat16 or float16, the block's output; rows a
            fixed number of elements apart are read in place, other strides
            are copied
        residual: the residual stream, of x's shape and type, or None (0)
        gate: (dim,) like the weights, or of x's shape and type, or None (1)
        post_weight, weight: (dim,) of x's type or float32, or None (1); they
            and a gate of (dim,) have one type
        scale: factor of the block's part
        eps: >= 0
        post_norm: whether x is normalised; if not, post_rstd is 1

    Returns (y, h, post_rstd, rstd): y, the new residual stream, and h, the next
    block's input, of x's shape and type; post_rstd and rstd are float32 of
    shape x.shape[:-1], as :func:`residual_norm_grad` takes them.  Sums are held
    in 32 bits, and h is made of y before its rounding.  So are squares: a row of
    x whose elements pass some 1e19 has an infinite mean square and adds nothing
    to y, a row of y that passes it has an h of 0; with an eps of 0 rows below some
    1e-19 have none.
    """
    x = _floats(x, "x")
    gate, post_weight, weight, kind, by_row = _block_inputs(x, gate, post_weight, weight, post_norm)
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0")
    if residual is not None:
        residual = _like(residual, "residual", x)
    y = _out(None, x.shape, x.dtype, x)
    h = torch.empty_like(y)
    post_rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(post_rstd)
    dim = x.shape[-1]
    x, rows, stride = _rows(x)
    residual, residual_stride, residual_at = _row_args(residual)
    gate, gate_stride, gate_at = _row_args(gate) if by_row else (gate, 0, _address(gate))
    _call("sporder_residual_norm", x, _TYPES[x.dtype], _TYPES[kind], rows, dim, stride,
          x.data_ptr(), residual_stride, residual_at, int(by_row), gate_stride, gate_at,
          _address(post_weight), _address(weight), float(scale), float(eps), int(bool(post_norm)),
          dim, y.data_ptr(), dim, h.data_ptr(), post_rstd.data_ptr(), rstd.data_ptr())
    return y, h, post_rstd, rstd


def residual_norm_grad(grad_y, grad_h, x, y, post_rstd, rstd, gate=None, post_weight=None,
                       weight=None, *, scale=1.0, post_norm=True):
    """Gradients of :func:`residual_norm`.

    Arguments:
        grad_y, grad_h: the gradients by y and h, of x's shape and type; either
            may be None (0)
        x, gate, post_weight, weight, scale, post_norm: as in the forward call
        y, post_rstd, rstd: as it returned them

    Returns (dx, dresidual, dgate, dpost_weight, dweight), None for what was
    not given (dresidual is returned always); each has its tensor's type.  Sums over the
    rows are held in 32 bits in an order that depends on the sizes and the
    inputs' types, strides and alignment: the same call gives the same bits
    from run to run.
    """
    x = _floats(x, "x")
    gate, post_weight, weight, kind, by_row = _block_inputs(x, gate, post_weight, weight, post_norm)
    y = _like(y, "y", x)
    if grad_y is not None:
        grad_y = _like(grad_y, "grad_y", x)
    if grad_h is not None:
        grad_h = _like(grad_h, "grad_h", x)
    for t, name in ((post_rstd, "post_rstd"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 \
                or t.shape != x.shape[:-1] or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name} must be the contiguous float32 tensor that residual_norm "
                             f"returned, of shape {tuple(x.shape[:-1])} on {x.device}")
    dx = _out(None, x.shape, x.dtype, x)
    dresidual = torch.empty_like(dx)
    dgate = None
    if gate is not None:
        dgate = torch.empty_like(dx) if by_row else torch.empty_like(gate)
    dpost = None if post_weight is None else torch.empty_like(post_weight)
    dweight = None if weight is None else torch.empty_like(weight)
    dim = x.shape[-1]
    x, rows, stride = _rows(x)
    y, _, y_stride = _rows(y)
    grad_y, dy_stride, dy_at = _row_args(grad_y)
    grad_h, dh_stride, dh_at = _row_args(grad_h)
    gate, gate_stride, gate_at = _row_args(gate) if by_row else (gate, 0, _address(gate))
    size = 0
    if not by_row and gate is not None or dpost is not None or dweight is not None:
        size = _lib.load().sporder_residual_norm_grad_work_bytes(rows, dim)
    work = x.new_empty(size, dtype=torch.uint8) if size else None
    _call("sporder_residual_norm_grad", x, _TYPES[x.dtype], _TYPES[kind], rows, dim, dy_stride,
          dy_at, dh_stride, dh_at, stride, x.data_ptr(), y_stride, y.data_ptr(),
          post_rstd.data_ptr(), rstd.data_ptr(), int(by_row), gate_stride, gate_at,
          _address(post_weight), _address(weight), float(scale), int(bool(post_norm)), dim,
          dx.data_ptr(), dim, dresidual.data_ptr(), dim, _address(dgate), _address(dpost),
          _address(dweight), _address(work), size)
    return dx, dresidual, dgate, dpost, dweight


def _one_pass(dtype, dim, classes):
    """Whether the loss takes any number of rows in one pass."""
    for most, floats, halves in ((48, 512, 512), (64, 384, 512), (96, 256, 512), (128, 192, 384),
                                 (192, 128, 256)):
        if classes <= most:
            return 8 <= dim <= (floats if dtype == torch.float32 else halves)
    return False


def _loss_inputs(x, weight, targets, bias):
    """(x of two dimensions, its stride, weight, its stride, targets, bias)."""
    x = _floats(x, "x")
    weight = _floats(weight, "weight")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > 65536:
        raise ValueError("x must have a last dimension of 1 to 65536 elements")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be a (classes, {x.shape[-1]}) tensor")
    if weight.dtype != x.dtype:
        raise TypeError("weight must have x's type")
    _same_device(weight, x, "weight")
    targets = _as_tensor(targets, "targets")
    if not targets.is_cuda:
        raise TypeError("targets must be a GPU tensor")
    if targets.dtype not in _TOKEN_BITS:
        raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
    _same_device(targets, x, "targets")
    if targets.shape != x.shape[:-1]:
        raise ValueError("targets must have the shape of x without its last dimension")
    if bias is not None:
        bias = _floats(bias, "bias")
        if bias.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"bias must have x's type or float32, got {bias.dtype}")
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"bias must have shape ({weight.shape[0]},)")
        _same_device(bias, x, "bias")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    classes, rows = weight.shape[0], targets.numel()
    if classes > 2**25:
        raise ValueError("at most 2^25 classes")
    if (rows > 2**23 - 256 or rows * classes > 2**37) and not _one_pass(x.dtype, x.shape[-1], classes):
        raise ValueError("at most 2^23 - 256 rows and 2^37 logits over so many classes and elements a row")
    x, _, x_stride = _rows(x)
    weight, _, weight_stride = _rows(weight)
    targets = targets if targets.is_contiguous() else targets.contiguous()
    return x, x_stride, weight, weight_stride, targets, bias


@functools.lru_cache(maxsize=256)
def _loss_work(name, kind, rows, dim, classes, x_stride, x_end, weight_stride, weight_end):
    """Bytes of scratch, a function of sizes, strides and the addresses' alignment to
    16 bytes alone (asking the library takes 1.2 us of a call's 18)."""
    return getattr(_lib.load(), name)(kind, rows, dim, classes, x_stride, 4096 + x_end,
                                      weight_stride, 4096 + weight_end)


def _ignored(ignore_index):
    ignore_index = int(ignore_index)
    if not -(2**63) <= ignore_index < 2**63:
        raise ValueError("ignore_index must fit 64 bits")
    return ignore_index


def linear_cross_entropy(x, weight, targets, bias=None, *, ignore_index=-100):
    """Softmax cross entropy of the logits z = x weight^T + bias, which are
    never kept: lse = log sum exp z, loss = lse - z[target], by row.

    Arguments:
        x: (..., dim) float32, bfloat16 or float16; rows a fixed number of
            elements apart are read in place, other strides are copied
        weight: (classes, dim) of x's type
        targets: int32 or int64 of shape x.shape[:-1]
        bias: (classes,) of x's type or float32, or None; -inf leaves a class out
        ignore_index: rows with this target have loss and lse 0 and are not read

    Returns (loss, lse, sums): loss and lse float32 of the targets' shape (NaN
    for a target that is neither a class nor ignored), sums float32 (2,) of the
    losses' sum and the number of rows that are not ignored.  At most 2^23 - 256
    rows and 2^37 logits (more over up to 48 classes of 8 to 512 elements, 64 of
    384, 96 of 256, 128 of 192 or 192 of 128; of 16-bit types 96 of 512, 128 of
    384 or 192 of 256), 2^25 classes and 65536 elements a row.  The gradients
    take the same sizes.

    Sums are held in 32 bits.  float32 products have operands of 22 bits: a term
    is within 2^-21 of itself, and within some 2^-38 of the product of its rows'
    largest elements; a row that holds an infinity gives NaN, and elements past
    some 1e33 may pass 32 bits on the way.
    """
    x, x_stride, weight, weight_stride, targets, bias = _loss_inputs(x, weight, targets, bias)
    ignore_index = _ignored(ignore_index)
    rows, (classes, dim) = targets.numel(), weight.shape
    loss = x.new_empty(targets.shape, dtype=torch.float32)
    lse = torch.empty_like(loss)
    sums = x.new_empty(2, dtype=torch.float32)
    kind, x_at, weight_at = _TYPES[x.dtype], x.data_ptr(), weight.data_ptr()
    sizes = (kind, rows, dim, classes, x_stride, x_at, weight_stride, weight_at)
    size = _loss_work("sporder_linear_cross_entropy_work_bytes", kind, rows, dim, classes,
                      x_stride, x_at % 16, weight_stride, weight_at % 16)
    work = x.new_empty(size, dtype=torch.uint8) if size else None
    _call("sporder_linear_cross_entropy", x, *sizes, _TYPES[x.dtype if bias is None else bias.dtype],
          _address(bias), _TOKEN_BITS[targets.dtype], targets.data_ptr(), ignore_index,
          loss.data_ptr(), lse.data_ptr(), sums.data_ptr(), _address(work), size)
    return loss, lse, sums


def linear_cross_entropy_grad(grad, x, weight, targets, lse, bias=None, *, ignore_index=-100,
                              dtype=None, loss=None):
    """Gradients of :func:`linear_cross_entropy` by x, weight and bias.

    Arguments:
        grad: the gradient by the losses, float32 of the targets' shape or of
            one element for all rows
        x, weight, targets, bias, ignore_index: as in the forward call
        lse: as it returned it
        dtype: weight's type (default) or float32, the type of weight's gradient
        loss: as the forward call returned it, or None; with it the target's g is
            made of the loss rather than of lse, whose rounding is more than all
            of it for rows that are sure of their target

    Returns (dx, dweight, dbias), dbias None without a bias.  The logits are
    made again, a piece of the rows and classes at a time, so that scratch is at
    most some 4 GB beside weight packed, its gradient in 32 bits and 40 bytes a
    row; rows that are ignored, or whose target is no class, have no gradient.  g = grad (exp(z - lse) -
    [target]) keeps 11 bits or more in its products with weight and x (22 for
    float32; nothing below 2^-38 of grad), weight's and x's elements nothing
    below 2^-40 of their column's largest, in dweight times the largest grad;
    sums are held in 32 bits.  The same call gives the same bits
    from run to run.
    """
    x, x_stride, weight, weight_stride, targets, bias = _loss_inputs(x, weight, targets, bias)
    ignore_index = _ignored(ignore_index)
    rows, (classes, dim) = targets.numel(), weight.shape
    for t, name in ((grad, "grad"), (lse, "lse"), (loss, "loss")):
        if t is None and name == "loss":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or not t.is_cuda:
            raise TypeError(f"{name} must be a float32 GPU tensor")
        _same_device(t, x, name)
        if name != "grad" and t.shape != targets.shape:
            raise ValueError(f"{name} must have the targets' shape")
    if grad.shape != targets.shape and grad.numel() != 1:
        raise ValueError("grad must have the targets' shape or one element")
    if dtype is None:
        dtype = weight.dtype
    elif dtype not in (weight.dtype, torch.float32):
        raise ValueError("dtype must be weight's type or float32")
    lse = lse if lse.is_contiguous() else lse.contiguous()
    if loss is not None and not loss.is_contiguous():
        loss = loss.contiguous()
    one = grad.numel() == 1 or all(s == 0 for s in grad.stride())
    if not one and not grad.is_contiguous():
        grad = grad.contiguous()
    dx = x.new_empty((*targets.shape, dim))
    dweight = weight.new_empty(weight.shape, dtype=dtype)
    dbias = None if bias is None else torch.empty_like(bias)
    sizes = (x_stride, x.data_ptr(), weight_stride, weight.data_ptr())
    size = _loss_work("sporder_linear_cross_entropy_grad_work_bytes", _TYPES[x.dtype], rows, dim,
                      classes, x_stride, x.data_ptr() % 16, weight_stride,
                      weight.data_ptr() % 16)
    work = x.new_empty(size, dtype=torch.uint8) if size else None
    _call("sporder_linear_cross_entropy_grad_of_loss", x, _TYPES[x.dtype], rows, dim, classes,
          0 if one else 1, grad.data_ptr(), *sizes,
          _TYPES[x.dtype if bias is None else bias.dtype], _address(bias),
          _TOKEN_BITS[targets.dtype], targets.data_ptr(), ignore_index, lse.data_ptr(),
          _address(loss), dim, dx.data_ptr(), _TYPES[dtype], dim, dweight.data_ptr(), _address(dbias),
          _address(work), size)
    return dx, dweight, dbias
