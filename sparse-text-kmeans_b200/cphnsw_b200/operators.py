"""Operators around the index, on ``torch`` tensors in device memory.

What a program that learns the vectors it indexes needs beside the index: rows of an embedding table and their gradient
(``embedding_lookup``, ``embedding_grad``), the loss that trains a student on a teacher's top scores and its gradient
(``distill_loss``, ``distill_loss_and_grad``; the lists are what ``exact_search_dev`` returns, distances negated), and products
of 8-bit vectors (``quantize_rows``, ``int8_matmul``), which score queries against a whole base set at a byte a coordinate.

Every call runs on the current torch stream of its tensors' device, returns without waiting, and takes its outputs and its
workspace from torch's allocator; a tensor that another stream has written or will reuse is the caller's to synchronise, as
with torch's own operations.  No autograd graph is recorded: the gradients are calls of their own.  While gradients are
recorded a tensor that requires one is therefore refused (``detach()`` it, or call under ``torch.no_grad()``), except as
the logits of ``distill_loss_and_grad``, whose gradient that call returns (``logits.backward(grad)`` goes on from
there).  A tensor given as ``out`` counts as changed in place.  Matrices may have any row stride (0 for a broadcast
row); where the elements of a row are not next to one another a contiguous copy is made.  Wrong arguments raise
``ValueError`` before anything is launched.  ``check_operator_status`` waits for the device and raises if a kernel gave
up a bounded wait.
"""
import ctypes as C

_TYPES = {}   # torch dtype -> element type of the C header
_IDS = {}     # torch dtype -> bytes of an id
_torch = None
_fn = {}      # the library's functions, by their names without prefix
_raw_stream = None
_current_device = None
_changed = None  # of a tensor: its values are others than autograd may have kept


def _bind():
    """Loads torch and the library once; with argument types set, plain integers can be passed."""
    global _torch, _raw_stream, _current_device, _changed
    import torch

    from . import load_library
    lib = load_library()
    p, u, i, w, f = C.c_void_p, C.c_uint64, C.c_int, C.c_uint32, C.c_float
    for name, args in {
        "embedding_lookup_dev": (p, i, u, u, u, p, w, u, f, p, u, p),
        "embedding_grad_dev": (p, w, u, p, i, u, f, p, i, u, u, u, i, p, u, p),
        "quantize_rows_dev": (p, i, u, u, u, p, u, p, p),
        "int8_matmul_dev": (p, u, p, u, p, u, p, u, u, p, i, u, p, u, p),
        "distill_loss_dev": (p, i, u, u, u, p, w, u, p, u, u, f, p, p),
        "distill_loss_and_grad_dev": (p, i, u, u, u, p, w, u, p, u, u, f, p, p, p, u, p, u, p),
        "embedding_grad_workspace": (u, u, u), "int8_matmul_workspace": (p, u, u, p, u, u, u), "distill_workspace": (u, u),
        "operator_status": (),
    }.items():
        fn = getattr(lib, "cphnsw_b200_" + name)
        fn.argtypes = args
        if name.endswith("_workspace"):
            fn.restype = u
        _fn[name] = fn
    _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    _IDS.update({torch.int32: 4, torch.int64: 8})
    # (the stream's address without a Stream object around it, which takes 2 us to make)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
    _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    _changed = torch.autograd.graph.increment_version
    _torch = torch


def _device(*tensors, differentiable=None):
    """The index of the tensors' one device.  What the caller would lose a gradient of is refused, but for ``differentiable``."""
    if _torch is None:
        _bind()
    dev = None
    for t in tensors:
        if not isinstance(t, _torch.Tensor) or not t.is_cuda:
            raise ValueError("expected torch tensors in device memory")
        at = t.get_device()
        if dev is None:
            dev = at
        elif at != dev:
            raise ValueError("tensors on several devices")
        if t.requires_grad and t is not differentiable and _torch.is_grad_enabled():
            raise ValueError("a tensor that requires a gradient: no graph is recorded here; pass t.detach(), or call under torch.no_grad()")
    return dev


def _call(dev, name, *args):
    """The library's function on the device's current stream."""
    if dev == _current_device():
        rc = _fn[name](*args, _raw_stream(dev))
    else:
        with _torch.cuda.device(dev):
            rc = _fn[name](*args, _raw_stream(dev))
    if rc:
        from . import _check
        _check(rc)


def _matrix(t, what, dtypes=None):
    """(the matrix, its rows, their length, the distance of one from the next; of a single row, its length)"""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError("%s: expected a matrix" % what)
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError("%s: element type %s is not supported" % (what, t.dtype))
    n, d = shape
    stride, step = t.stride()
    if step != 1 and d > 1:
        t = t.contiguous()
        stride = d
    return t, n, d, stride if n > 1 else d or 1


def _output(out, shape, dtype, dev, what, replaced=None):
    """The caller's output, after a look at it.  One that requires a gradient cannot be written to while gradients are recorded,
    unless it is ``replaced``, and no leaf."""
    if not isinstance(out, _torch.Tensor) or not out.is_cuda or out.get_device() != dev or tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError("%s: out must be %s of shape %s on the inputs' device" % (what, dtype, tuple(shape)))
    if shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError("%s: out needs elements of a row next to one another" % what)
    if out.requires_grad and _torch.is_grad_enabled() and (out is not replaced or out.is_leaf):
        raise ValueError("%s: out requires a gradient" % what)
    return out


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=_torch.uint8) if nbytes else None


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _stride(t):
    """Row stride; of a single row, its length."""
    n, d = t.shape
    return t.stride(0) if n > 1 else d or 1


def _flat_ids(ids, what):
    if ids.dtype not in _IDS:
        raise ValueError("%s: ids must be int32 or int64" % what)
    return ids if ids.is_contiguous() else ids.contiguous()


def embedding_lookup(table, ids, scale=1.0, out=None):
    """``scale * table[ids]``: [*ids.shape, dim] in the table's type.  An id outside the table (a search's "no node" is -1 as
    int32) gives zeros."""
    dev = _device(table, ids)
    table, rows, dim, table_stride = _matrix(table, "embedding_lookup", _TYPES)
    ids = _flat_ids(ids, "embedding_lookup")
    n = ids.numel()
    shape = (*ids.shape, dim)
    given = out is not None
    if given:
        _output(out, shape, table.dtype, dev, "embedding_lookup")
        try:
            stride = _stride(out if out.dim() == 2 else out.view(n, dim))
        except RuntimeError:
            raise ValueError("embedding_lookup: out needs rows at one distance from one another") from None
    else:
        out = table.new_empty(shape)
        stride = dim
    _call(dev, "embedding_lookup_dev", table.data_ptr(), _TYPES[table.dtype], rows, dim, table_stride, ids.data_ptr(), _IDS[ids.dtype], n, scale,
          out.data_ptr(), stride)
    if given:
        _changed(out)
    return out


def embedding_grad(ids, grad, rows, scale=1.0, dtype=None, out=None, accumulate=False):
    """The gradient of ``embedding_lookup``'s table, [rows, dim]: ``scale`` times the sum of the rows of ``grad`` ([*ids.shape,
    dim]) over the places that hold an id.  ``dtype``: fp32 or grad's (the default).  With ``accumulate`` it is added to
    ``out``.  The same input gives the same bits."""
    dev = _device(ids, grad)
    ids = _flat_ids(ids, "embedding_grad")
    n = ids.numel()
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError("embedding_grad: grad must have the ids' shape and a last dimension")
    dim = grad.shape[-1]
    grad, _, _, grad_stride = _matrix(grad if grad.dim() == 2 else grad.reshape(n, dim), "embedding_grad", _TYPES)
    if accumulate and out is None:
        raise ValueError("embedding_grad: accumulate needs out")
    if dtype is None:
        dtype = grad.dtype if out is None else out.dtype
    if dtype not in _TYPES:
        raise ValueError("embedding_grad: element type %s is not supported" % dtype)
    rows = int(rows)
    if rows < 1:
        raise ValueError("embedding_grad: need rows >= 1")
    given = out is not None
    out = _output(out, (rows, dim), dtype, dev, "embedding_grad") if given else grad.new_empty((rows, dim), dtype=dtype)
    ws = _workspace(_fn["embedding_grad_workspace"](n, rows, dim), grad)
    _call(dev, "embedding_grad_dev", ids.data_ptr(), _IDS[ids.dtype], n, grad.data_ptr(), _TYPES[grad.dtype], grad_stride, scale, out.data_ptr(),
          _TYPES[dtype], rows, dim, _stride(out), int(bool(accumulate)), _ptr(ws), 0 if ws is None else ws.numel())
    if given:
        _changed(out)
    return out


def quantize_rows(x):
    """Rows to 8 bits with a scale each: (q int8 [n, dim], scale float32 [n]), ``scale = max|x| / 127`` (by the rounded
    1 / 127) and ``q = x / scale`` rounded to the nearest, ties to even.  q's rows start at multiples of 16 bytes, as
    ``int8_matmul`` likes them."""
    dev = _device(x)
    x, n, dim, stride = _matrix(x, "quantize_rows", _TYPES)
    pitch = (dim + 15) // 16 * 16
    q = x.new_empty((n, pitch), dtype=_torch.int8)
    if pitch != dim:
        q = q[:, :dim]
    scale = x.new_empty(n, dtype=_torch.float32)
    _call(dev, "quantize_rows_dev", x.data_ptr(), _TYPES[x.dtype], n, dim, stride, q.data_ptr(), pitch, scale.data_ptr())
    return q, scale


def _scales(t, n, what):
    if t.dtype != _torch.float32 or t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s: expected float32[%d]" % (what, n))
    return t if t.is_contiguous() else t.contiguous()


def int8_matmul(a, a_scale, b, b_scale, dtype=None, out=None):
    """``(a @ b.T) * a_scale[:, None] * b_scale[None, :]``: a int8 [m, k], b int8 [n, k], the sums exact, the result [m, n] of
    type ``dtype`` (bfloat16 unless said, or out's)."""
    dev = _device(a, a_scale, b, b_scale)
    a, m, k, sa = _matrix(a, "int8_matmul", (_torch.int8,))
    b, n, d, sb = _matrix(b, "int8_matmul", (_torch.int8,))
    if d != k:
        raise ValueError("int8_matmul: rows of %d and %d values" % (k, d))
    a_scale, b_scale = _scales(a_scale, m, "int8_matmul"), _scales(b_scale, n, "int8_matmul")
    if dtype is None:
        dtype = _torch.bfloat16 if out is None else out.dtype
    if dtype not in _TYPES:
        raise ValueError("int8_matmul: element type %s is not supported" % dtype)
    given = out is not None
    if given:
        stride = _stride(_output(out, (m, n), dtype, dev, "int8_matmul"))
    else:
        out, stride = a.new_empty((m, n), dtype=dtype), n or 1
    pa, pb = a.data_ptr(), b.data_ptr()
    ws = None
    if (pa | pb | sa | sb) % 16:
        ws = _workspace(_fn["int8_matmul_workspace"](pa, sa, m, pb, sb, n, k), a)
    _call(dev, "int8_matmul_dev", pa, sa, a_scale.data_ptr(), m, pb, sb, b_scale.data_ptr(), n, k, out.data_ptr(), _TYPES[dtype], stride,
          _ptr(ws), 0 if ws is None else ws.numel())
    if given:
        _changed(out)
    return out


def _lists(logits, ids, teacher, what):
    """(each with its rows, their length and distance, as _matrix tells)"""
    logits = _matrix(logits, what, _TYPES)
    shape = ids.shape
    if len(shape) != 2 or ids.dtype not in _IDS or teacher.shape != shape or shape[0] != logits[1]:
        raise ValueError("%s: ids (int32 or int64) and teacher must be [n, top] for logits [n, rows]" % what)
    if teacher.dtype not in _TYPES:
        raise ValueError("%s: element type %s is not supported" % (what, teacher.dtype))
    return logits, _matrix(ids, what), _matrix(teacher if teacher.dtype == _torch.float32 else teacher.to(_torch.float32), what)


def distill_loss(logits, ids, teacher, temperature=1.0):
    """The distillation loss of every row, float32 [n]: ``T^2 KL(softmax(teacher / T) || softmax(logits / T))`` with the
    teacher's logits given at the places ``ids`` [n, top] of a row only (ids outside the row: empty places)."""
    dev = _device(logits, ids, teacher)
    (logits, n, rows, stride), (ids, _, top, ids_stride), (teacher, _, _, teacher_stride) = _lists(logits, ids, teacher, "distill_loss")
    loss = teacher.new_empty(n)
    _call(dev, "distill_loss_dev", logits.data_ptr(), _TYPES[logits.dtype], n, rows, stride, ids.data_ptr(), _IDS[ids.dtype], ids_stride,
          teacher.data_ptr(), teacher_stride, top, temperature, loss.data_ptr())
    return loss


def distill_loss_and_grad(logits, ids, teacher, weight=None, temperature=1.0, out=None):
    """``distill_loss`` and the gradient of its sum, weighted by ``weight`` float32 [n] (1 unless given), with respect to the
    logits, in their type: (loss [n], grad [n, rows]).  ``out`` may be ``logits`` itself."""
    student = logits
    tensors = (logits, ids, teacher) if weight is None else (logits, ids, teacher, weight)
    dev = _device(*tensors, differentiable=student)
    (logits, n, rows, stride), (ids, _, top, ids_stride), (teacher, _, _, teacher_stride) = _lists(logits, ids, teacher, "distill_loss_and_grad")
    if weight is not None:
        weight = _scales(weight, n, "distill_loss_and_grad")
    if out is None:
        grad, grad_stride = logits.new_empty((n, rows)), rows or 1
    else:
        grad = _output(out, (n, rows), logits.dtype, dev, "distill_loss_and_grad", replaced=student)
        grad_stride = _stride(grad)
    loss = teacher.new_empty(n)
    ws = _workspace(_fn["distill_workspace"](n, top), teacher)
    _call(dev, "distill_loss_and_grad_dev", logits.data_ptr(), _TYPES[logits.dtype], n, rows, stride, ids.data_ptr(), _IDS[ids.dtype],
          ids_stride, teacher.data_ptr(), teacher_stride, top, temperature, _ptr(weight), loss.data_ptr(), grad.data_ptr(), grad_stride,
          _ptr(ws), 0 if ws is None else ws.numel())
    if out is not None:
        _changed(out)
    return loss, grad


def check_operator_status(device=0):
    """Waits for the device; raises ``CPHNSWError`` if an operator's kernel has given up a bounded wait since the last check."""
    if _torch is None:
        _bind()
    from . import _check
    with _torch.cuda.device(device):
        _check(_fn["operator_status"]())
