"""What the row operators refuse, on the host and before any device call: shapes,
types, strides, alignments, sizes, workspaces and overlaps, through Python and
through the C ABI. The addresses are never followed."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import powersparse_amd as ps
from powersparse_amd import _native
from powersparse_amd._native import Ids, Rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A, B, C, D = (k << 32 for k in (1, 2, 3, 4))  # addresses far from each other


def mat(at, rows, cols, dtype="float32", **more):
    return ps.DeviceArray(at, (rows, cols), dtype, **more)


def vec(at, n, dtype):
    return ps.DeviceArray(at, n, dtype)


def refused(text, f, *args, **kwargs):
    with pytest.raises(ValueError, match=text):
        f(*args, **kwargs)


def test_every_declared_symbol_is_exported_and_bound():
    text = open(os.path.join(ROOT, "include", "powersparse_rows.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"^\s*[A-Za-z_][\w\s\*]*?\b(ps_\w+)\s*\(", text, re.M)))
    _native.libs()
    out = subprocess.run(["nm", "-D", "--defined-only", _native.HIP_LIB_PATH],
                         capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if line.strip()}
    assert len(names) >= 12 and not [n for n in names if n not in exported]
    assert set(names) == {n for n, _, _ in _native.ROWS_API}


def test_device_array():
    refused("dtype", ps.DeviceArray, A, 4, "float64")
    refused("one or two dimensions", ps.DeviceArray, A, (2, 2, 2))
    refused("one or two dimensions", ps.DeviceArray, A, (-1,))
    refused("row stride", ps.DeviceArray, A, (2, 8), ld=7)
    refused("row stride", ps.DeviceArray, A, 8, ld=9)

    class Buffer:
        ptr, nbytes = A, 64

    refused("too small", ps.DeviceArray, Buffer(), 17)
    refused("too small", ps.DeviceArray, Buffer(), (2, 4), ld=13)
    assert ps.DeviceArray(Buffer(), (2, 4), ld=12).ptr == A
    assert ps.DeviceArray(Buffer(), 8, "float16", offset=24).ptr == A + 48
    refused("too small", ps.DeviceArray, Buffer(), 8, "float16", offset=25)


def test_tensors_on_the_host_are_refused():
    host = torch.zeros((4, 4))
    ids = torch.zeros(4, dtype=torch.int64)
    refused("table is not in device memory", ps.EmbeddingLookup, host, ids, host)
    refused("ids is not in device memory", ps.EmbeddingLookup, mat(A, 4, 4), ids, mat(B, 4, 4))
    refused("not a device array", ps.EmbeddingLookup, [1.0], ids, host)
    refused("gradient 0 is not in device memory", ps.GradientList, [host])
    refused("workspace is not in device memory", ps.EmbeddingGrad, vec(C, 4, "int32"),
            mat(A, 4, 4), mat(B, 4, 4), torch.zeros(1 << 20, dtype=torch.uint8))


def test_lookup():
    def call(table=None, ids=None, out=None):
        ps.EmbeddingLookup(table or mat(A, 9, 8), ids or vec(B, 4, "int64"), out or mat(C, 4, 8))

    refused("out is not ids x table columns", call, out=mat(C, 5, 8))
    refused("out is not ids x table columns", call, out=mat(C, 4, 9))
    refused("overlap", call, out=mat(A + 64, 4, 8))
    refused("overlap", call, table=mat(A, 9, 8, ld=32), out=mat(A + 16, 4, 8, ld=32))
    refused("element type int32", call, table=mat(A, 9, 8, "int32"))
    refused("ids: element type float32", call, ids=vec(B, 4, "float32"))
    refused("not a matrix", call, out=vec(C, 32, "float32"))
    refused("misaligned", call, table=mat(A + 2, 9, 8))
    refused("misaligned", call, ids=vec(B + 4, 4, "int64"))
    refused("null data", call, table=mat(0, 9, 8))
    refused("null data", call, ids=vec(0, 4, "int64"))
    refused("bad shape", call, table=mat(A, 9, 0), out=mat(C, 4, 0))


def test_lookup_grad():
    work = vec(D, ps.embedding_grad_workspace_bytes(40, 8, 9), "uint8")

    def call(ids=None, dy=None, grad=None, work=work):
        ps.EmbeddingGrad(ids or vec(B, 40, "int32"), dy or mat(A, 40, 8), grad or mat(C, 9, 8),
                         work)

    refused("grad_out is not ids x grad columns", call, dy=mat(A, 41, 8))
    refused("grad_out is not ids x grad columns", call, grad=mat(C, 9, 7))
    refused("overlap", call, grad=mat(A, 9, 8))
    refused("workspace too small", call, work=vec(D, work.shape[0] - 1, "uint8"))
    refused("workspace too small or misaligned", call, work=vec(D + 8, 1 << 20, "uint8"))
    refused("workspace too small", call, work=vec(0, work.shape[0], "uint8"))
    refused("out of range", ps.embedding_grad_workspace_bytes, -1, 8, 9)
    refused("out of range", ps.embedding_grad_workspace_bytes, 8, 0, 9)
    refused("out of range", ps.embedding_grad_workspace_bytes, 8, 8, 1 << 31)


def test_expert_sort():
    work = vec(D, ps.expert_sort_workspace_bytes(40, 5), "uint8")

    def call(ids=None, order=None, position=None, offsets=None, work=work):
        ps.ExpertSort(ids or mat(A, 20, 2, "int64"), order or vec(B, 40, "int32"),
                      position or mat(B + 4096, 20, 2, "int32"), offsets or vec(C, 6, "int32"),
                      work)

    refused("1 to 1024 experts", call, offsets=vec(C, 1, "int32"))
    refused("1 to 1024 experts", call, offsets=vec(C, 1026, "int32"))
    refused("order has 39 elements where 40", call, order=vec(B, 39, "int32"))
    refused("position has 42 elements", call, position=mat(B, 21, 2, "int32"))
    refused("offsets: element type int64", call, offsets=vec(C, 6, "int64"))
    refused("ids is not contiguous", call, ids=mat(A, 20, 2, "int64", ld=3))
    refused("workspace too small", call, work=vec(D, work.shape[0] - 1, "uint8"))
    refused("null output", call, order=vec(0, 40, "int32"))
    refused("1 to 1024 experts", ps.expert_sort_workspace_bytes, 40, 1025)


def test_dispatch_and_combine():
    x, xs, at = mat(A, 20, 8), mat(B, 40, 8), mat(C, 20, 2, "int32")
    w = mat(C + 4096, 20, 2)
    refused("41 slots do not divide among 20", ps.ExpertDispatch, x, vec(C, 41, "int32"), xs)
    refused("differ in type or width", ps.ExpertDispatch, x, at, mat(B, 40, 8, "float16"))
    refused("differ in type or width", ps.ExpertDispatch, x, at, mat(B, 40, 9))
    refused("overlap", ps.ExpertDispatch, x, at, mat(A + 32, 40, 8))
    refused("null positions", ps.ExpertDispatch, x, mat(0, 20, 2, "int32"), xs)
    refused("1 to 1024 slots", ps.ExpertDispatch, x, mat(C, 20, 1025, "int32"), xs)
    refused("weights has 41 elements", ps.ExpertCombine, xs, at, vec(D, 41, "float32"), x)
    refused("weights: element type float16", ps.ExpertCombine, xs, at, mat(D, 20, 2, "float16"), x)
    refused("differ in type or width", ps.ExpertCombine, mat(B, 40, 7), at, w, x)
    refused("overlap", ps.ExpertCombine, mat(A, 40, 8), at, w, x)
    refused("overlap", ps.ExpertDispatchGrad, mat(A, 40, 8), at, x)
    dw = mat(D, 20, 2)
    refused("differ in type, width or rows", ps.ExpertCombineGrad, x, xs, at, w, mat(D, 39, 8), dw)
    refused("overlaps an input", ps.ExpertCombineGrad, x, xs, at, w, xs, dw)
    refused("dweights has 20 elements", ps.ExpertCombineGrad, x, xs, at, w, mat(D, 40, 8),
            mat(D, 20, 1))


def test_column_ranges_of_one_matrix_that_overlap():
    """x and xs in the rows of one buffer, some columns in common."""
    for off in (1, 7, 25, 31, 33):
        refused("overlap", ps.ExpertDispatch, mat(A, 20, 8, ld=32), mat(C, 20, 1, "int32"),
                mat(A + 4 * off, 20, 8, ld=32))
        refused("overlap", ps.ExpertDispatch, mat(A + 640, 1, 8), mat(C, 1, 1, "int32"),
                mat(A + 4 * off, 20, 8, ld=32))
    refused("overlap", ps.ExpertDispatch, mat(A, 1, 8), mat(C, 1, 1, "int32"), mat(A + 4, 1, 8))


def test_gradient_list():
    g = vec(A, 100, "float32")
    refused("outs: one for each", ps.GradientList, [g], [])
    refused("output 0 has 99 elements", ps.GradientList, [g], [vec(B, 99, "float32")])
    refused("gradient 0: element type int32", ps.GradientList, [vec(A, 4, "int32")])
    refused("tensor 0: null data", ps.GradientList, [vec(0, 4, "float32")])
    refused("tensor 1: misaligned", ps.GradientList, [g, vec(B + 2, 4, "float32")])
    refused("overlaps its output", ps.GradientList, [g], [vec(A + 4, 100, "float32")])
    refused("overlaps its output", ps.GradientList, [g], [vec(A, 100, "float16")])
    h = vec(A + 400, 100, "float32")
    refused("listed twice", ps.GradientList, [g, h, g])
    refused("listed twice", ps.GradientList, [h, vec(A + 4, 100, "float32")])
    refused("overlaps another", ps.GradientList, [g, h], [vec(B, 100, "float32"), g])
    refused("overlaps another", ps.GradientList, [g, h], [vec(B, 100, "float32"),
                                                          vec(B + 396, 100, "float32")])
    hip = _native.hip()
    assert hip.ps_grad_norm(None, 1.0, A, None) == _native.PS_ERR_INVALID
    assert hip.ps_clip_grads(None, 1.0, 1.0, A, None) == _native.PS_ERR_INVALID
    assert hip.ps_clip_grad_norm(None, 1.0, 1.0, A, None) == _native.PS_ERR_INVALID
    hip.ps_grad_list_destroy(None)


def test_c_abi():
    """What Python cannot pass."""
    hip = _native.hip()
    ok, ids = Rows(A, 4, 8, 8, 0), Ids(B, 4, 0)
    out = Rows(C, 4, 8, 8, 0)
    bad = [(None, ids, out), (ok, None, out), (ok, ids, None), (Rows(A, 4, 8, 8, 3), ids, out),
           (Rows(A, 4, 8, 8, -1), ids, out), (Rows(A, -1, 8, 8, 0), ids, out),
           (Rows(A, 4, 8, 7, 0), ids, out), (Rows(A, 1 << 40, 8, 1 << 20, 0), ids, out),
           (Rows(A, 4, (1 << 24) + 1, 1 << 25, 0), ids, out), (ok, Ids(B, 4, 2), out),
           (ok, Ids(B, -1, 0), out), (ok, Ids(B, (1 << 30) + 1, 0), out)]
    for t, i, o in bad:
        assert hip.ps_embedding_lookup(t, i, 1.0, o, None) == _native.PS_ERR_INVALID
        assert _native.hip().ps_last_error()


# where the sorts' tiles and digits and the gradient's chunks change
COUNTS = sorted({n + d for n in [1, 16, 1024, 4096, 65536, 1 << 30] +
                 [4 * 4096 << k for k in range(8)] + [192 * 1024 << k for k in range(4)] +
                 [1024 * 4096] for d in (-8, -1, 0, 1, 8) if 0 <= n + d <= 1 << 30})
COLS = [1, 4, 7, 8, 9, 64, 336, 1023, 1024, 4096, 8191, 1 << 20, 1 << 24]
ROWS = sorted({r + d for r in (0, 2, 511, 1023, 1 << 17, 1 << 20, 1 << 25, (1 << 31) - 3)
               for d in (0, 1)})
EXPERTS = [1, 2, 3, 4, 63, 64, 511, 1023, 1024]


def never_less(size, *axes):
    """size() never shrinks along any axis: neighbours on the grid are enough."""
    def walk(fixed, rest):
        if rest:
            for v in rest[0]:
                yield from walk(fixed + (v,), rest[1:])
        else:
            yield fixed
    for place, axis in enumerate(axes):
        others = axes[:place] + axes[place + 1:]
        for fixed in walk((), others):
            sizes = [size(*fixed[:place], v, *fixed[place:]) for v in axis]
            for k in range(1, len(axis)):
                assert sizes[k] >= sizes[k - 1], (place, fixed, axis[k - 1:k + 1],
                                                  sizes[k - 1:k + 1])


def test_a_workspace_for_the_largest_call_does_for_smaller_ones():
    never_less(ps.embedding_grad_workspace_bytes, COUNTS, COLS, ROWS)
    never_less(ps.expert_sort_workspace_bytes, COUNTS, EXPERTS)


def test_what_is_written_overlaps_nothing_else():
    """Kernels take the places that they write from ids and workspaces, so nothing written may
    be anything else that the call reads or writes, by a single byte."""
    def work_bytes(n):
        return vec(D, n, "uint8")

    table, ids, out = mat(A, 9, 8), vec(B, 40, "int64"), mat(C, 40, 8)
    at_end = C + 40 * 8 * 4
    refused("overlap", ps.EmbeddingLookup, table, vec(C, 40, "int64"), out)
    refused("overlap", ps.EmbeddingLookup, table, vec(at_end - 8, 40, "int64"), out)
    refused("overlap", ps.EmbeddingLookup, table, vec(C - 40 * 8 + 8, 40, "int64"), out)

    n = ps.embedding_grad_workspace_bytes(40, 8, 9)
    work, grad, dy = work_bytes(n), mat(A, 9, 8), mat(C, 40, 8)
    refused("overlap", ps.EmbeddingGrad, vec(A, 40, "int64"), dy, grad, work)
    for at in (A, B, C):  # the workspace on the gradient, the ids, the rows
        refused("overlap", ps.EmbeddingGrad, ids, dy, grad, vec(at, n, "uint8"))
    refused("overlap", ps.EmbeddingGrad, ids, dy, grad, vec(at_end - 16, n, "uint8"))

    n = ps.expert_sort_workspace_bytes(40, 5)
    order, position, offsets = vec(B, 40, "int32"), vec(C, 40, "int32"), vec(A + 4096, 6, "int32")
    ids, work = vec(A, 40, "int32"), work_bytes(n)
    whole = [ids, order, position, offsets, work]
    for i in range(5):
        for j in range(5):
            if i != j:
                moved = list(whole)
                was = whole[i]
                moved[i] = vec(whole[j].ptr, was.shape[0], was.dtype)
                refused("overlap", ps.ExpertSort, *moved)

    x, xs, at = mat(A, 20, 8), mat(B, 40, 8), mat(C, 20, 2, "int32")
    w, dw = mat(C + 4096, 20, 2), mat(C + 8192, 20, 2)
    refused("overlap", ps.ExpertDispatch, x, mat(B + 36, 20, 2, "int32"), xs)
    refused("overlap", ps.ExpertCombine, xs, mat(A + 36, 20, 2, "int32"), w, x)
    refused("overlap", ps.ExpertCombine, xs, at, mat(A + 36, 20, 2), x)
    dys = mat(D, 40, 8)
    for f, where in ((0, "position"), (1, "weights"), (2, "dweights")):
        args = [x, xs, at, w, dys, dw]
        args[(2, 3, 5)[f]] = mat(D + 36, 20, 2, "int32" if f == 0 else "float32")
        refused("overlap", ps.ExpertCombineGrad, *args)
    for taken in (A, B, C, C + 4096):  # dy, ys, positions, weights
        refused("overlap", ps.ExpertCombineGrad, x, xs, at, w, dys, mat(taken, 20, 2))


def test_flat_arrays_that_reach_from_between_rows_into_them():
    """Columns 24 to 31 of a matrix's rows are not its own: positions there are refused from
    the first column that is."""
    for first in (23, 25, 31):
        refused("overlap", ps.ExpertDispatch, mat(A, 8, 24),
                mat(B + 4 * first, 8, 1, "int32"), mat(B, 20, 24, ld=32))


def test_slots_of_another_shape():
    """(tokens, top_k) arrays of as many elements that belong to another number of tokens."""
    x, xs = mat(A, 4, 8), mat(B, 16, 8)
    w, dw = mat(C + 4096, 4, 4), mat(C + 8192, 4, 4)
    for shape in ((8, 2), (2, 8), (16, 1), (1, 16)):
        wrong = mat(C, *shape, "int32")
        text = f"position: {shape[0]} x {shape[1]} slots for 4 tokens"
        refused(text, ps.ExpertDispatch, x, wrong, xs)
        refused(text, ps.ExpertCombine, xs, wrong, w, x)
        refused(text, ps.ExpertDispatchGrad, xs, wrong, x)
        refused(text, ps.ExpertCombineGrad, x, xs, wrong, w, mat(D, 16, 8), dw)
    at = mat(C, 4, 4, "int32")
    for shape in ((8, 2), (2, 8)):
        other = mat(C + 4096, *shape)
        text = f"weights: {shape[0]} x {shape[1]} slots for 4 tokens"
        refused("^" + text, ps.ExpertCombine, xs, at, other, x)
        refused("^" + text, ps.ExpertCombineGrad, x, xs, at, other, mat(D, 16, 8), dw)
        refused("^d" + text, ps.ExpertCombineGrad, x, xs, at, w, mat(D, 16, 8), other)


def test_slots_as_a_list_or_of_a_batch():
    """One dimension, or any shape whose leading dimensions hold the tokens."""
    class Slots:  # a tensor as far as its description goes
        is_cuda, dtype = True, "int32"

        def __init__(self, *shape):
            self.shape = shape

        def is_contiguous(self):
            return True

        def numel(self):
            n = 1
            for s in self.shape:
                n *= s
            return n

        def stride(self):
            return tuple(Slots(*self.shape[k + 1:]).numel() for k in range(len(self.shape)))

        def data_ptr(self):
            return C

    from powersparse_amd import rows
    for shape in ((16,), (4, 4), (2, 2, 4), (4, 1, 4), (1, 4, 4), (4, 4, 1), (4, 2, 2)):
        assert rows._top_k(Slots(*shape), 4) == (C, 4)
    assert rows._top_k(Slots(4), 4) == (C, 1) == rows._top_k(Slots(4, 1), 4)
    assert rows._top_k(Slots(8, 1), 1) == (C, 8)  # one token: every shape is its
    assert rows._top_k(Slots(0, 3), 0)[0] == C
    for shape in ((2, 4, 2), (8, 2, 1), (0, 4), (4, 0), (15,), (3, 4)):
        refused("position", rows._top_k, Slots(*shape), 4)


def test_tensors_of_another_device(monkeypatch):
    """Where there are several devices, every tensor's is compared with the current one."""
    from powersparse_amd import rows

    class Tensor:
        is_cuda = True

        def __init__(self, at, shape, dtype="float32", device=0):
            self.shape, self.dtype, self.at, self.device = tuple(shape), dtype, at, device

        def get_device(self):
            return self.device

        def is_contiguous(self):
            return True

        def numel(self):
            n = 1
            for s in self.shape:
                n *= s
            return n

        def stride(self):
            return tuple(Tensor(0, self.shape[k + 1:]).numel() for k in range(len(self.shape)))

        def data_ptr(self):
            return self.at

    class List:
        handle, device = 1 << 40, 0

        def get_device(self):
            return self.device

    called = []
    monkeypatch.setattr(rows, "_several", None)
    monkeypatch.setattr(rows, "_count_devices", lambda: 2)
    monkeypatch.setattr(rows, "_current_device", lambda: 0)

    class Library:
        def __getattr__(self, name):
            return lambda *a: called.append(name) or 0

    monkeypatch.setattr(rows, "_hip", Library())
    table, out, dw = Tensor(A, (4, 8)), Tensor(B, (4, 8)), Tensor(B + 4096, (4, 1))
    ids, at = Tensor(C, (4,), "int32"), Tensor(C + 4096, (4, 1), "int32")
    off, w = Tensor(C + 8192, (6,), "int32"), Tensor(D, (4, 1))
    work = Tensor(D + 4096, (99,), "uint8")
    norm, glist = Tensor(A + 4096, (1,)), List()
    calls = [(ps.EmbeddingLookup, (table, ids, out)), (ps.EmbeddingGrad, (ids, table, out, work)),
             (ps.ExpertSort, (ids, Tensor(A, (4,), "int32"), at, off, work)),
             (ps.ExpertDispatch, (table, at, out)), (ps.ExpertCombine, (table, at, w, out)),
             (ps.ExpertDispatchGrad, (table, at, out)),
             (ps.ExpertCombineGrad, (table, out, at, w, Tensor(D + (1 << 20), (4, 8)), dw)),
             (ps.GradNorm, (glist, norm)), (ps.ClipGrads, (glist, 1.0, norm)),
             (ps.ClipGradNorm, (glist, 1.0, norm))]
    for f, args in calls:
        f(*args)  # all on the current device
        assert len(called) == 1
        called.clear()
        for x in args:
            if isinstance(x, (Tensor, List)):
                x.device = 1
                refused("on device 1, the current one is 0", f, *args)
                x.device = 0
    for x in (table, out):
        x.device = 1
        refused("on device 1, the current one is 0", ps.GradientList, [table], [out])
        x.device = 0
    assert not called
    # arrays that name no device are taken as they are
    ps.EmbeddingLookup(mat(A, 4, 8), vec(C, 4, "int32"), mat(B, 4, 8))
    assert called == ["ps_embedding_lookup"]
    assert rows._several is True
    # one device: found out once, and never asked again
    monkeypatch.setattr(rows, "_several", None)
    monkeypatch.setattr(rows, "_count_devices", lambda: 1)
    table.device = 1
    ps.EmbeddingLookup(table, ids, out)
    assert rows._several is False


def test_sizes_beyond_the_c_types():
    """ctypes keeps the low bits of larger numbers: 2^32 + 8 experts would be 8."""
    for experts in ((1 << 32) + 8, -(1 << 32) + 8, (1 << 31)):
        refused("out of range", ps.expert_sort_workspace_bytes, 40, experts)
    for n in ((1 << 64) + 8, -(1 << 64) + 8):
        refused("out of range", ps.expert_sort_workspace_bytes, n, 8)
        for sizes in ((n, 8, 9), (8, n, 9), (8, 8, n)):
            refused("out of range", ps.embedding_grad_workspace_bytes, *sizes)
    many = (1 << 32) + 2
    refused("1 to 1024 slots", ps.ExpertDispatch, mat(A, 1, 8), vec(1 << 40, many, "int32"),
            mat(B, 4, 8))
    refused("1 to 1024 experts", ps.ExpertSort, vec(A, 4, "int32"), vec(B, 4, "int32"),
            vec(C, 4, "int32"), vec(1 << 40, many, "int32"), vec(D, 1 << 20, "uint8"))


def test_padding_beyond_64_bits(monkeypatch):
    """No id is such a number: it is passed on as one that no row has."""
    from powersparse_amd import rows
    passed = []

    class Library:
        def ps_embedding_grad(self, *args):
            passed.append(ctypes.c_longlong(args[3]).value)
            return 0

    monkeypatch.setattr(rows, "_hip", Library())
    for padding in ((1 << 64) + 3, (1 << 63) + 3, 3, 0, -1, -(1 << 63), -(1 << 64) + 3):
        ps.EmbeddingGrad(vec(B, 40, "int32"), mat(A, 40, 8), mat(C, 9, 8),
                         vec(D, 1 << 20, "uint8"), padding_idx=padding)
        assert passed.pop() == padding if 0 <= padding < 9 else not 0 <= passed.pop() < 9
