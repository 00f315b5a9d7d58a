"""Row operators on the device: embedding lookup and its gradient, tokens sorted by expert
and back with their gradients, and the norm and clipping of many gradient tensors
(include/powersparse_rows.h).

Arrays are in the current device's memory: DeviceArray (a DeviceBuffer or raw pointer with
a shape and a type) or any tensor object with data_ptr, shape, stride, dtype and is_cuda,
such as torch's; tensors that say they are on another device are refused. Matrices are
row-major with any row stride; element types are float32, float16 and bfloat16. Every call
checks shapes, types and sizes on the host, enqueues its kernels on `stream` (a Stream, a
tensor library's stream, a raw handle, or None: the null stream) and returns without
synchronising: arrays and workspaces must stay alive, and be written by nothing else, until
the stream has passed the call. Wrong arguments raise ValueError.
"""
import ctypes

from . import _native
from ._native import Ids, Rows


class _Library:
    """libpowersparse_hip.so's entry points, looked up once each (loaded on first use)."""

    def __getattr__(self, name):
        f = getattr(_native.hip(), name)
        setattr(self, name, f)
        return f


_hip = _Library()

_DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2}
_ID_TYPES = {"int32": 0, "int64": 1}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8, "uint8": 1}


class DeviceArray:
    """A one- or two-dimensional array in device memory: `data` (DeviceBuffer, another
    object with a `ptr`, or a device address), `shape`, `dtype` ("float32", "float16",
    "bfloat16", "int32", "int64", "uint8"), `ld` the row stride in elements (default:
    contiguous) and `offset` where it begins, in elements."""

    def __init__(self, data, shape, dtype="float32", ld=None, offset=0):
        if dtype not in _BYTES:
            raise ValueError(f"dtype must be one of {sorted(_BYTES)}")
        shape = (shape,) if isinstance(shape, int) else tuple(int(s) for s in shape)
        if len(shape) not in (1, 2) or min(shape) < 0 or offset < 0:
            raise ValueError("a DeviceArray has one or two dimensions")
        self.shape, self.dtype, self.data = shape, dtype, data
        self.ld = int(ld) if ld is not None else shape[-1]
        if len(shape) == 1 and self.ld != shape[0] or self.ld < shape[-1]:
            raise ValueError("row stride shorter than a row")
        size = _BYTES[dtype]
        elements = 0 if 0 in shape else (self.ld * (shape[0] - 1) + shape[1] if len(shape) == 2
                                         else shape[0])
        nbytes = getattr(data, "nbytes", None)
        if nbytes is not None and (offset + elements) * size > nbytes:
            raise ValueError("the buffer is too small for the array")
        base = data.ptr if hasattr(data, "ptr") else int(data or 0)
        self.ptr = (base or 0) + offset * size


# Type codes by name, and by a tensor library's dtype objects as they are met.
_row_codes = dict(_DTYPES)
_id_codes = dict(_ID_TYPES)
_names = {}


def _dtype_name(dtype):
    name = _names.get(dtype)
    if name is None:
        name = _names[dtype] = str(dtype).rsplit(".", 1)[-1]
        for names, codes in ((_DTYPES, _row_codes), (_ID_TYPES, _id_codes)):
            if name in names:
                codes[dtype] = names[name]
    return name


def _described(x, name):
    """(address, shape, strides, dtype) of an array."""
    if type(x) is DeviceArray:
        return x.ptr, x.shape, (x.ld, 1) if len(x.shape) == 2 else (1,), x.dtype
    try:
        if x.is_cuda:
            return x.data_ptr(), x.shape, x.stride(), x.dtype
    except (AttributeError, TypeError):
        raise ValueError(f"{name}: not a device array") from None
    raise ValueError(f"{name} is not in device memory")


def _code(dtype, codes, name, wanted):
    """The type code of a dtype that `codes` does not hold yet."""
    said = _dtype_name(dtype)
    if dtype not in codes:
        raise ValueError(f"{name}: element type {said} is not {wanted}")
    return codes[dtype]


def _rows(x, name):
    """The ps_rows of a matrix."""
    try:  # a tensor as it mostly is; anything else, and what is refused, below
        if x.is_cuda:
            (rows, cols), (ld, step) = x.shape, x.stride()
            if step == 1 and rows > 1:
                return Rows(x.data_ptr(), rows, cols, ld, _row_codes[x.dtype])
    except (AttributeError, KeyError, TypeError, ValueError):
        pass
    ptr, shape, stride, dtype = _described(x, name)
    code = _row_codes.get(dtype)
    if code is None:
        code = _code(dtype, _row_codes, name, "float32, float16 or bfloat16")
    if len(shape) != 2:
        raise ValueError(f"{name} is not a matrix")
    rows, cols = shape
    ld, step = stride
    if step != 1 and cols > 1 and rows:
        raise ValueError(f"{name}: elements of a row are not contiguous")
    return Rows(ptr, rows, cols, ld if rows > 1 else cols, code)


def _contiguous(shape, stride, name):
    """The element count of a contiguous array of any shape."""
    n = 1
    for s, d in zip(reversed(shape), reversed(stride)):
        if d != n and s > 1 and 0 not in shape:
            raise ValueError(f"{name} is not contiguous")
        n *= s
    return n


def _flat(x, name, dtypes, count=None):
    """Address, element count and dtype name of a contiguous array of any shape."""
    try:
        if x.is_cuda and x.is_contiguous() and _names[x.dtype] in dtypes:
            n = x.numel()
            if count is None or n == count:
                return x.data_ptr(), n, _names[x.dtype]
    except (AttributeError, KeyError, TypeError):
        pass
    ptr, shape, stride, dtype = _described(x, name)
    said = _dtype_name(dtype)
    if said not in dtypes:
        raise ValueError(f"{name}: element type {said} is not {' or '.join(dtypes)}")
    n = _contiguous(shape, stride, name)
    if count is not None and n != count:
        raise ValueError(f"{name} has {n} elements where {count} are needed")
    return ptr, n, said


def _ids(x, name="ids"):
    try:
        if x.is_cuda and x.is_contiguous():
            return Ids(x.data_ptr(), x.numel(), _id_codes[x.dtype])
    except (AttributeError, KeyError, TypeError):
        pass
    ptr, shape, stride, dtype = _described(x, name)
    code = _id_codes.get(dtype)
    if code is None:
        code = _code(dtype, _id_codes, name, "int32 or int64")
    return Ids(ptr, _contiguous(shape, stride, name), code)


def _space(x, name="workspace"):
    """Address and bytes of a workspace: a DeviceBuffer or a contiguous array."""
    try:
        if x.is_cuda and x.is_contiguous():
            return x.data_ptr(), x.numel() * _BYTES[_names[x.dtype]]
    except (AttributeError, KeyError, TypeError):
        pass
    if hasattr(x, "nbytes") and hasattr(x, "ptr") and not isinstance(x, DeviceArray):
        return x.ptr, x.nbytes
    ptr, n, dtype = _flat(x, name, _BYTES)
    return ptr, n * _BYTES[dtype]


def _stream(stream):
    if stream is None or type(stream) is int:
        return stream
    if hasattr(stream, "ptr"):
        return stream.ptr
    return int(getattr(stream, "cuda_stream", stream))


def _fit(n, most):
    """n within [-1, most], so that ctypes, which keeps the low bits of larger numbers, hands
    over one that is as far out of range."""
    return max(-1, min(int(n), most))


_INT, _LONG = (1 << 31) - 1, (1 << 63) - 1


def _call(status):
    if status:
        from . import _hip_call
        _hip_call(status)


def _count_devices():
    from . import device_count
    try:
        return device_count()
    except RuntimeError:  # none: every call fails at its launch
        return 0


def _current_device():
    d = ctypes.c_int()
    _call(_native.hip().ps_get_device(ctypes.byref(d)))
    return d.value


# Whether there are several devices (None: not known yet): calls then look where their arrays
# are. With one device nothing is asked.
_several = None


def _check_devices(*arrays):
    """Refuses tensors that say they are on another device than the current one, whose kernels
    would follow their addresses."""
    global _several
    if _several is None:
        _several = _count_devices() > 1
    if not _several:
        return
    here = _current_device()
    for x in arrays:
        try:
            at = x.get_device()
        except AttributeError:
            continue
        if at >= 0 and at != here:
            raise ValueError(f"an array is on device {at}, the current one is {here}")


# --------------------------------------------------------------- embedding

def EmbeddingLookup(table, ids, out, scale=1.0, stream=None):
    """out[i] = scale * table[ids[i]]; zeros for ids outside the table. `ids` (int32 or
    int64, any shape) are taken in order; out has one row for each. table and out may differ
    in type."""
    if _several is not False:
        _check_devices(table, ids, out)
    _call(_hip.ps_embedding_lookup(_rows(table, "table"), _ids(ids), scale, _rows(out, "out"),
                                   _stream(stream)))


def embedding_grad_workspace_bytes(count, cols, table_rows):
    """Workspace of EmbeddingGrad for `count` ids, rows of `cols` and a table of `table_rows`,
    or for fewer of any of them."""
    n = _hip.ps_embedding_grad_workspace_bytes(_fit(count, _LONG), _fit(cols, _LONG),
                                                _fit(table_rows, _LONG))
    if not n:
        raise ValueError("embedding_grad_workspace_bytes: sizes out of range")
    return n


def EmbeddingGrad(ids, grad_out, grad_table, workspace, scale=1.0, padding_idx=-1,
                  accumulate=False, stream=None):
    """grad_table[v] = scale * sum of grad_out[i] over the i with ids[i] = v, zeros for rows
    without ids; accumulate=True adds to grad_table instead. Ids outside the table and
    `padding_idx` take no part. The sum's order is fixed: the same bits every time."""
    if _several is not False:
        _check_devices(ids, grad_out, grad_table, workspace)
    ptr, nbytes = _space(workspace)
    _call(_hip.ps_embedding_grad(
        _ids(ids), _rows(grad_out, "grad_out"), scale, _fit(padding_idx, _LONG), bool(accumulate),
        _rows(grad_table, "grad_table"), ptr, nbytes, _stream(stream)))


# ----------------------------------------------------------------- experts

def expert_sort_workspace_bytes(slots, experts):
    """Workspace of ExpertSort for `slots` ids (tokens * top_k) and `experts` experts, or for
    fewer of either."""
    n = _hip.ps_expert_sort_workspace_bytes(_fit(slots, _LONG), _fit(experts, _INT))
    if not n:
        raise ValueError("expert_sort_workspace_bytes: sizes out of range (1 to 1024 experts)")
    return n


def ExpertSort(ids, order, position, offsets, workspace, stream=None):
    """Stable sort of the slots of `ids` (tokens x top_k experts) by expert: `order` the slots
    by expert, dropped ones (id outside the experts) last; `position` each slot's place in
    `order`, -1 for dropped ones; `offsets` (experts + 1) where each expert's slots begin.
    All int32."""
    if _several is not False:
        _check_devices(ids, order, position, offsets, workspace)
    slots = _ids(ids)
    at, count, _ = _flat(offsets, "offsets", ("int32",))
    ptr, nbytes = _space(workspace)
    _call(_hip.ps_expert_sort(
        slots, _fit(count - 1, _INT), _flat(order, "order", ("int32",), slots.count)[0],
        _flat(position, "position", ("int32",), slots.count)[0], at, ptr, nbytes,
        _stream(stream)))


def _slots(x, name, dtype, tokens, count=None):
    """Address of a value per slot, `count` of them, and slots per token. The leading
    dimensions of its shape hold the tokens, unless it has one dimension only: an array of as
    many elements for other tokens would be read across them."""
    try:
        if x.is_cuda and x.is_contiguous():
            rows, top_k = x.shape
            if rows == tokens and 0 < top_k <= _INT and rows and \
                    count in (None, rows * top_k) and _names[x.dtype] == dtype:
                return x.data_ptr(), top_k
    except (AttributeError, KeyError, TypeError, ValueError):
        pass
    ptr, n, _ = _flat(x, name, (dtype,), count)
    if tokens == 0:
        return ptr, 1
    if n == 0 or n % tokens:
        raise ValueError(f"{name}: {n} slots do not divide among {tokens} tokens")
    shape, leading = x.shape, 1
    if len(shape) > 1:
        for s in shape:
            if leading >= tokens:
                break
            leading *= s
        if leading != tokens:
            raise ValueError(f"{name}: {' x '.join(str(s) for s in shape)} slots for {tokens} "
                             "tokens")
    return ptr, _fit(n // tokens, _INT)


def _top_k(position, tokens):
    """Address of the positions and slots per token."""
    return _slots(position, "position", "int32", tokens)


def ExpertDispatch(x, position, xs, stream=None):
    """xs[position[t, k]] = x[t]: every token's row to its slots' places. Rows of xs that no
    position names are left alone, positions outside xs are skipped. `position` is (tokens,
    top_k), a flat list of the same, or any shape whose leading dimensions hold the tokens;
    weights below likewise."""
    if _several is not False:
        _check_devices(x, position, xs)
    src = _rows(x, "x")
    ptr, top_k = _top_k(position, src.rows)
    _call(_hip.ps_expert_dispatch(src, ptr, top_k, _rows(xs, "xs"), _stream(stream)))


def ExpertCombine(ys, position, weights, y, stream=None):
    """y[t] = sum over k of weights[t, k] * ys[position[t, k]] (float32 weights; None: ones);
    positions outside ys are skipped."""
    if _several is not False:
        _check_devices(ys, position, weights, y)
    out = _rows(y, "y")
    ptr, top_k = _top_k(position, out.rows)
    w = None
    if weights is not None:
        w = _slots(weights, "weights", "float32", out.rows, out.rows * top_k)[0]
    _call(_hip.ps_expert_combine(_rows(ys, "ys"), ptr, w, top_k, out, _stream(stream)))


def ExpertDispatchGrad(dxs, position, dx, stream=None):
    """The gradient of ExpertDispatch: dx[t] = sum over k of dxs[position[t, k]]."""
    ExpertCombine(dxs, position, None, dx, stream)


def ExpertCombineGrad(dy, ys, position, weights, dys, dweights, stream=None):
    """The gradients of ExpertCombine: dys[position[t, k]] = weights[t, k] * dy[t] and
    dweights[t, k] = <dy[t], ys[position[t, k]]>, 0 for dropped slots. Rows of dys that no
    position names are left alone."""
    if _several is not False:
        _check_devices(dy, ys, position, weights, dys, dweights)
    src = _rows(dy, "dy")
    ptr, top_k = _top_k(position, src.rows)
    n = src.rows * top_k
    _call(_hip.ps_expert_combine_grad(
        src, _rows(ys, "ys"), ptr, _slots(weights, "weights", "float32", src.rows, n)[0], top_k,
        _rows(dys, "dys"), _slots(dweights, "dweights", "float32", src.rows, n)[0],
        _stream(stream)))


# --------------------------------------------------------------- gradients

def _spans(arrays, what):
    """Addresses, element counts and type codes of contiguous arrays."""
    n = max(len(arrays), 1)
    data, counts, types = (ctypes.c_void_p * n)(), (ctypes.c_longlong * n)(), (ctypes.c_int * n)()
    for i, x in enumerate(arrays):
        code = _row_codes.get(getattr(x, "dtype", None))
        if code is not None and type(x) is not DeviceArray and x.is_cuda and x.is_contiguous():
            data[i], counts[i], types[i] = x.data_ptr(), x.numel(), code  # some hundred at a time
        else:
            data[i], counts[i], said = _flat(x, f"{what} {i}", _DTYPES)
            types[i] = _DTYPES[said]
    return data, counts, types


class GradientList:
    """The gradient tensors of a model (contiguous arrays of any shape and of float32,
    float16 or bfloat16) and where their clipped values go: `outs`, one of the same size for
    each, or None for in place. Made once while the tensors stay where they are, as making it
    uploads and waits for the device (37 tensors 42 us, 291 146 us); calls on one list must
    not overlap. Keeps the tensors alive. Closing it, or losing it, waits for nothing."""

    def __init__(self, grads, outs=None):
        self._h = None
        self._keep = (list(grads), list(outs) if outs is not None else None)
        grads, outs = self._keep
        if outs is not None and len(outs) != len(grads):
            raise ValueError("outs: one for each gradient")
        if _several is not False:
            _check_devices(*grads, *(outs or ()))
        n = len(grads)
        data, counts, types = _spans(grads, "gradient")
        to = to_types = None
        if outs is not None:
            to, sizes, to_types = _spans(outs, "output")
            for i in range(n):
                if sizes[i] != counts[i]:
                    raise ValueError(f"output {i} has {sizes[i]} elements where {counts[i]} "
                                     "are needed")
        h = ctypes.c_void_p()
        _call(_hip.ps_grad_list_create(n, data, counts, types, to, to_types, ctypes.byref(h)))
        self._h = h.value
        self._device = _current_device()

    def get_device(self):
        """The device it was made on."""
        return self._device

    @property
    def handle(self):
        if not self._h:
            raise ValueError("the gradient list is closed")
        return self._h

    def close(self):
        if self._h:
            _hip.ps_grad_list_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def GradNorm(grads, norm, grad_scale=1.0, stream=None):
    """norm (one float32 on the device) = the 2-norm of grad_scale * g over a GradientList."""
    if _several is not False:
        _check_devices(grads, norm)
    _call(_hip.ps_grad_norm(grads.handle, grad_scale, _flat(norm, "norm", ("float32",), 1)[0],
                            _stream(stream)))


def ClipGrads(grads, max_norm, norm, grad_scale=1.0, stream=None):
    """g * grad_scale * min(1, max_norm / (norm + 1e-6)) with a given norm, e.g. one that the
    ranks of a job have put together."""
    if _several is not False:
        _check_devices(grads, norm)
    _call(_hip.ps_clip_grads(grads.handle, max_norm, grad_scale,
                             _flat(norm, "norm", ("float32",), 1)[0], _stream(stream)))


def ClipGradNorm(grads, max_norm, norm, grad_scale=1.0, stream=None):
    """GradNorm and ClipGrads in one call: norm receives the norm before clipping."""
    if _several is not False:
        _check_devices(grads, norm)
    _call(_hip.ps_clip_grad_norm(grads.handle, max_norm, grad_scale,
                                 _flat(norm, "norm", ("float32",), 1)[0], _stream(stream)))
