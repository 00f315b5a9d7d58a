"""What layer norm, the router and AdamW refuse, on the host and before any device call, through
Python and through the C ABI, and their workspace sizes. The addresses are never followed."""
import ctypes
import math

import numpy as np
import pytest
import torch

import powersparse_amd as ps
from powersparse_amd import _native
from powersparse_amd._native import AdamWOptions, AdamWTensor, Rows

A, B, C, D, E, G = (k << 32 for k in (1, 2, 3, 4, 5, 6))  # addresses far from each other


def mat(at, rows, cols, dtype="float32", **more):
    return ps.DeviceArray(at, (rows, cols), dtype, **more)


def vec(at, n, dtype="float32"):
    return ps.DeviceArray(at, n, dtype)


def refused(text, f, *args, **kwargs):
    with pytest.raises(ValueError, match=text):
        f(*args, **kwargs)


def test_layer_norm():
    def call(x=None, w=None, b=None, y=None, mean=None, rstd=None, eps=1e-5):
        ps.LayerNorm(x or mat(A, 9, 8), w, b, y or mat(C, 9, 8), mean, rstd, eps=eps)

    refused("differ in shape", call, y=mat(C, 8, 8))
    refused("differ in shape", call, y=mat(C, 9, 7))
    refused("weight is not one row of x's columns", call, w=vec(B, 7))
    refused("bias is not one row of x's columns", call, b=vec(B, 9, "float16"))
    refused("weight is not a vector", call, w=mat(B, 1, 8))
    refused("weight: element type int32", call, w=vec(B, 8, "int32"))
    refused("mean has 8 elements where 9", call, mean=vec(B, 8))
    refused("rstd: element type float16", call, rstd=vec(B, 9, "float16"))
    refused("misaligned mean or rstd", call, mean=vec(B + 2, 9))
    refused("misaligned", call, w=vec(B + 2, 8))
    refused("null data", call, y=mat(0, 9, 8))
    for eps in (-1e-9, float("nan")):
        refused("eps is not a number", call, eps=eps)
    refused("overlap", call, y=mat(A, 9, 8))
    refused("overlap", call, y=mat(A + 4, 9, 8))
    refused("overlap", call, w=vec(C + 4, 8))
    refused("overlap", call, b=vec(C + 9 * 32 - 4, 8))
    refused("overlap", call, mean=vec(C, 9))
    refused("overlap", call, mean=vec(B, 9), rstd=vec(B + 32, 9))
    refused("overlap", call, rstd=vec(A + 4, 9))
    refused("overlap", call, w=vec(B, 8), mean=vec(B + 28, 9))


def test_layer_norm_grad():
    n = ps.layer_norm_grad_workspace_bytes(9, 8)
    good = dict(dy=mat(A, 9, 8), x=mat(B, 9, 8), weight=vec(C, 8), mean=vec(C + 4096, 9),
                rstd=vec(C + 8192, 9), dx=mat(D, 9, 8), dweight=vec(E, 8), dbias=vec(E + 4096, 8),
                workspace=vec(G, n, "uint8"))

    def call(**other):
        ps.LayerNormGrad(**{**good, **other})

    refused("differ in shape", call, dy=mat(A, 8, 8))
    refused("differ in shape", call, dx=mat(D, 9, 9))
    refused("dx and x in type", call, dx=mat(D, 9, 8, "float16"))
    refused("dweight is not one row", call, dweight=vec(E, 7))
    refused("dbias is not one row", call, dbias=vec(E, 9))
    refused("null mean or rstd", call, mean=None)
    refused("null mean or rstd", call, rstd=None)
    refused("misaligned mean", call, rstd=vec(C + 1, 9))
    refused("workspace too small", call, workspace=vec(G, n - 1, "uint8"))
    refused("workspace too small or misaligned", call, workspace=vec(G + 4, n + 64, "uint8"))
    refused("workspace too small", call, workspace=None)
    refused("workspace too small", call, workspace=None, dweight=None)
    inputs, outputs = ("dy", "x", "weight", "mean", "rstd"), ("dx", "dweight", "dbias", "workspace")
    for o in outputs:
        for other in inputs + outputs:
            if o != other:
                x = good[o]
                moved = ps.DeviceArray(good[other].ptr, x.shape, x.dtype)
                refused("overlap", call, **{o: moved})
    for sizes in ((-1, 8), (8, 0), (8, (1 << 24) + 1), ((1 << 48) + 1, 8)):
        refused("out of range", ps.layer_norm_grad_workspace_bytes, *sizes)


def test_route():
    n = ps.expert_route_workspace_bytes(20, 5)
    good = dict(logits=mat(A, 20, 5), ids=mat(B, 20, 2, "int32"), weights=mat(C, 20, 2),
                counts=vec(D, 6, "int32"), loss=vec(D + 4096, 1), workspace=vec(G, n, "uint8"),
                mask=vec(E, 20, "uint8"))

    def call(**other):
        ps.ExpertRoute(**{**good, **other})

    refused("1 to 1024 experts", call, logits=mat(A, 20, 1025), counts=vec(D, 1026, "int32"))
    refused("as many slots a token as there are experts", call, ids=mat(B, 20, 6, "int32"),
            weights=mat(C, 20, 6))
    refused("ids: element type int64", call, ids=mat(B, 20, 2, "int64"))
    refused("weights has 20 elements", call, weights=mat(C, 20, 1))
    refused("10 x 4 slots for 20 tokens", call, ids=mat(B, 10, 4, "int32"))
    refused("counts has 5 elements", call, counts=vec(D, 5, "int32"))
    refused("loss has 2 elements", call, loss=vec(D, 2))
    refused("mask has 19 elements", call, mask=vec(E, 19, "uint8"))
    refused("mask: element type int32", call, mask=vec(E, 20, "int32"))
    refused("come together", call, loss=None)
    refused("come together", call, counts=None)
    refused("workspace too small", call, workspace=None)
    refused("workspace too small", call, workspace=vec(G, n - 1, "uint8"))
    refused("workspace too small or misaligned", call, workspace=vec(G + 8, n, "uint8"))
    refused("null ids or weights", call, ids=mat(0, 20, 2, "int32"))
    refused("misaligned output", call, weights=mat(C + 2, 20, 2))
    outputs = ("ids", "weights", "counts", "loss", "workspace")
    for o in outputs:
        for other in ("logits", "mask") + outputs:
            if o != other:
                x = good[o]
                moved = ps.DeviceArray(good[other].ptr, x.shape, x.dtype)
                refused("overlap", call, **{o: moved})
    for sizes in ((-1, 5), (20, 0), (20, 1025), ((1 << 30) + 1, 5)):
        refused("out of range", ps.expert_route_workspace_bytes, *sizes)


def test_route_grad():
    good = dict(logits=mat(A, 20, 5), ids=mat(B, 20, 2, "int32"), dweights=mat(C, 20, 2),
                counts=vec(D, 6, "int32"), dloss=vec(D + 4096, 1), dlogits=mat(E, 20, 5))

    def call(**other):
        ps.ExpertRouteGrad(**{**good, **other})

    refused("differ in type or shape", call, dlogits=mat(E, 20, 6))
    refused("differ in type or shape", call, dlogits=mat(E, 20, 5, "float16"))
    refused("dweights has 60 elements", call, dweights=mat(C, 20, 3))
    refused("needs the counts", call, counts=None)
    refused("null ids", call, ids=mat(0, 20, 2, "int32"))
    refused("misaligned input", call, dweights=mat(C + 2, 20, 2))
    for other in ("logits", "ids", "dweights", "counts", "dloss"):
        refused("overlaps an input", call, dlogits=ps.DeviceArray(good[other].ptr, (20, 5)))


def good_list(**other):
    n = 1000
    args = dict(params=[vec(A, n)], grads=[vec(B, n, "float16")], exp_avgs=[vec(C, n)],
                exp_avg_sqs=[vec(D, n)], copies=[vec(E, n, "bfloat16")])
    args.update(other)
    return args


def test_adamw_list():
    def call(**other):
        ps.AdamWList(**good_list(**other))

    refused("grads: one for each parameter", call, grads=[])
    refused("copies: one for each parameter", call, copies=[None, None])
    refused("weight_decay: one for each parameter", call, weight_decay=[0.1, 0.2])
    refused("gradient 0 has 999 elements", call, grads=[vec(B, 999)])
    refused("parameter 0: element type int32", call, params=[vec(A, 1000, "int32")])
    refused("exp_avg 0: element type float16", call, exp_avgs=[vec(C, 1000, "float16")])
    refused("exp_avg 0: element type uint8 is not float32", call, exp_avgs=[vec(C, 1000, "uint8")])
    refused("exp_avg_sq 0 has 1001", call, exp_avg_sqs=[vec(D, 1001)])
    refused("tensor 0: null data", call, grads=[vec(0, 1000)])
    refused("tensor 0: misaligned", call, exp_avgs=[vec(C + 2, 1000)])
    refused("tensor 0: weight decay is not", call, weight_decay=float("nan"))
    for decay in (1e300, [1e300], ["0.1"], [None]):
        refused("weight.decay (0 )?is not a number", call, weight_decay=decay)
    codes = dict(exp_avgs=[vec(C, 1000, "uint8")], exp_avg_sqs=[vec(D, 1000, "uint8")])
    refused("scales 0 has 7 elements where 8", call, scales=[vec(G, 7)], **codes)
    refused("exp_avg 0: element type float32", call, scales=[vec(G, 8)])
    refused("tensor 0: null data", call, scales=[vec(0, 8)], **codes)
    refused("tensor 0: misaligned", call, scales=[vec(G + 2, 8)], **codes)
    good = good_list()
    for name in ("params", "exp_avgs", "exp_avg_sqs", "copies"):
        for other in good:
            if other != name:
                x = good[name][0]
                for at in (0, 1000 * (4 if x.dtype == "float32" else 2) - 4):
                    moved = ps.DeviceArray(good[other][0].ptr - at, 1000, x.dtype)
                    refused("overlap", call, **{name: [moved]})
    refused("overlap", call, scales=[vec(A + 3996, 8)], **codes)
    two = {k: v + [ps.DeviceArray(v[0].ptr + (1 << 20), 1000, v[0].dtype)]
           for k, v in good.items()}
    two["exp_avgs"][1] = two["exp_avg_sqs"][0]
    refused("overlap, or a tensor is listed twice", ps.AdamWList, **two)


def test_adamw_c_abi():
    hip = _native.hip()
    bad = _native.PS_ERR_INVALID
    out = ctypes.c_void_p()

    def tensor(**other):
        t = AdamWTensor(param=A, grad=B, exp_avg=C, exp_avg_sq=D, scales=E, count=1000,
                        weight_decay=0.1)
        for k, v in other.items():
            setattr(t, k, v)
        return ctypes.byref(t)

    assert hip.ps_adamw_list_create(1, tensor(), 0, None) == bad
    assert hip.ps_adamw_list_create(-1, tensor(), 0, ctypes.byref(out)) == bad
    assert hip.ps_adamw_list_create(1, None, 0, ctypes.byref(out)) == bad
    for state in (1, 2, 4, -1):
        assert hip.ps_adamw_list_create(1, tensor(), state, ctypes.byref(out)) == bad
    for other in (dict(param_dtype=3), dict(grad_dtype=-1), dict(copy=G, copy_dtype=3),
                  dict(count=-1), dict(count=1 << 45), dict(weight_decay=float("inf")),
                  dict(exp_avg=None), dict(scales=None), dict(param=A + 1),
                  dict(exp_avg_sq=C + 999)):
        assert hip.ps_adamw_list_create(1, tensor(**other), 3, ctypes.byref(out)) == bad, other
        assert out.value is None
    hip.ps_adamw_list_destroy(None)
    o = AdamWOptions(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, grad_scale=1.0)
    assert hip.ps_adamw_step(None, ctypes.byref(o), None) == bad
    ok = Rows(A, 4, 8, 8, 0)
    for w in (Rows(B, 2, 8, 8, 0), Rows(B, 1, 8, 8, 3), Rows(B, 0, 8, 8, 0)):
        assert hip.ps_layer_norm(ok, w, None, 1e-5, Rows(C, 4, 8, 8, 0), None, None, None) == bad
    for top_k in (0, -1, 9):
        assert hip.ps_expert_route(ok, top_k, 1, None, B, C, None, None, None, 0, None) == bad
        assert hip.ps_expert_route_grad(ok, top_k, 1, B, C, None, None, Rows(D, 4, 8, 8, 0),
                                        None) == bad
    # 2^30 slots at most
    many = Rows(A, (1 << 29) + 1, 2, 2, 2)
    assert hip.ps_expert_route(many, 2, 1, None, 8 << 40, 9 << 40, None, None, None, 0, None) == bad


def test_workspaces_grow_with_every_argument():
    rows = sorted({max(0, n + d) for n in (0, 16, 512, 1024, 1 << 20, 1 << 24, 1 << 30)
                   for d in (-1, 0, 1)})
    cols = [1, 2, 7, 64, 1023, 4095, 4096, 4097, 8191, 65536, 1 << 18, (1 << 18) + 1, 1 << 20, 1 << 24]
    for axis in ([ps.layer_norm_grad_workspace_bytes(r, c) for c in cols] for r in rows):
        assert axis == sorted(axis)
    for axis in ([ps.layer_norm_grad_workspace_bytes(r, c) for r in rows] for c in cols):
        assert axis == sorted(axis)
    tokens, experts = [r for r in rows if r <= 1 << 30], [1, 2, 5, 63, 64, 65, 1023, 1024]
    for axis in ([ps.expert_route_workspace_bytes(t, e) for e in experts] for t in tokens):
        assert axis == sorted(axis)
    for axis in ([ps.expert_route_workspace_bytes(t, e) for t in tokens] for e in experts):
        assert axis == sorted(axis)


def test_state_blocks():
    assert [ps.state_blocks(n) for n in (0, 1, 256, 257, 1 << 33)] == [0, 1, 1, 2, 1 << 25]


def test_adamw_weight_decay_of_no_dimension():
    """A number in an array without dimensions is a number."""
    two = {k: v + [ps.DeviceArray(v[0].ptr + (1 << 20), 1000, v[0].dtype)]
           for k, v in good_list().items()}
    for value in (math.nan, 1e300):
        for number in (np.array(value), torch.tensor(value, dtype=torch.float64)):
            refused("weight.decay (0 )?is not a number", ps.AdamWList, weight_decay=number, **two)
    refused("weight_decay: one for each parameter", ps.AdamWList, weight_decay=np.zeros(3), **two)
    refused("tensor 1: weight decay is not", ps.AdamWList,
            weight_decay=torch.tensor([0.1, float("nan")]), **two)


def test_adamw_list_of_iterators():
    """What may be gone through once is taken like a list, as for gradient lists."""
    def call(**other):
        given = good_list(**other)
        ps.AdamWList(**{k: iter(v) for k, v in given.items()})

    refused("gradient 0 has 999 elements", call, grads=[vec(B, 999)])
    refused("grads: one for each parameter", call, grads=[])
    refused("copies: one for each parameter", call, copies=[None, None])
    refused("weight_decay: one for each parameter", call, weight_decay=[0.1, 0.2])
    codes = dict(exp_avgs=[vec(C, 1000, "uint8")], exp_avg_sqs=[vec(D, 1000, "uint8")])
    refused("scales 0 has 7 elements where 8", call, scales=[vec(G, 7)], **codes)
    refused("scales: one for each parameter", call, scales=[], **codes)
