"""What the layer norm and AdamW refuse, before any work is enqueued (runs without a GPU), and the AdamW plan's image."""
import ctypes

import pytest
import torch

from recommenders_amd import _lib
from recommenders_amd.models.deeprec.models.adamw import AdamW

lib = _lib.lib


def refused(rc, text, code=-1):
    assert rc == code, rc
    assert text in lib.xdfm_last_error().decode(), lib.xdfm_last_error()


def norm_fwd(**kw):
    a = dict(x=4096, xs=8, dtype=0, rows=2, cols=8, gamma=64, beta=64, eps=1e-5, act=0, y=8192, ys=8, stats=None)
    a.update(kw)
    return lib.xdfm_layer_norm_fwd(a["x"], a["xs"], a["dtype"], a["rows"], a["cols"], a["gamma"], a["beta"], a["eps"],
                                   a["act"], a["y"], a["ys"], a["stats"], None)


def norm_bwd(**kw):
    a = dict(x=4096, xs=8, dy=8192, dys=8, dtype=0, rows=2, cols=8, gamma=64, beta=64, stats=64, act=0, dx=16384, dxs=8,
             dg=64, db=64, ws=64)
    a.update(kw)
    return lib.xdfm_layer_norm_bwd(a["x"], a["xs"], a["dy"], a["dys"], a["dtype"], a["rows"], a["cols"], a["gamma"],
                                   a["beta"], a["stats"], a["act"], a["dx"], a["dxs"], a["dg"], a["db"], a["ws"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"), (dict(act=5), "activation"),
    (dict(act=-1), "activation"), (dict(rows=-1), "bad sizes"), (dict(cols=0), "bad sizes"), (dict(xs=7), "bad sizes"),
    (dict(ys=7), "bad sizes"), (dict(rows=1 << 62), "bad sizes"), (dict(cols=(1 << 30) + 1, xs=1 << 31, ys=1 << 31), "bad sizes"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(y=None), "null"), (dict(gamma=None), "null"),
    (dict(beta=None), "null"), (dict(x=4097), "misaligned"), (dict(y=8194), "misaligned"),
    (dict(dtype=1, x=4097), "misaligned"), (dict(y=4096, ys=9), "same stride"),
])
def test_layer_norm_forward_refuses(kw, text):
    refused(norm_fwd(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "element type"), (dict(act=5), "activation"), (dict(rows=-1), "bad sizes"), (dict(cols=-4), "bad sizes"),
    (dict(xs=7), "bad sizes"), (dict(dys=7), "bad sizes"), (dict(dxs=7), "bad sizes"), (dict(x=None), "null"),
    (dict(dy=None), "null"), (dict(dx=None), "null"), (dict(stats=None), "null"), (dict(gamma=None), "null"),
    (dict(dg=None), "null"), (dict(db=None), "null"), (dict(ws=None), "null"), (dict(rows=0, ws=None), "null"),
    (dict(ws=68), "misaligned"), (dict(dx=16385), "misaligned"), (dict(dx=8192, dxs=9), "same stride"),
    (dict(dx=4096, dxs=9), "same stride"),
])
def test_layer_norm_backward_refuses(kw, text):
    refused(norm_bwd(**kw), text)


def test_layer_norm_workspace():
    size = ctypes.c_size_t()
    refused(lib.xdfm_layer_norm_bwd_workspace_floats(4, 0, ctypes.byref(size)), "bad argument")
    refused(lib.xdfm_layer_norm_bwd_workspace_floats(-1, 4, ctypes.byref(size)), "bad argument")
    refused(lib.xdfm_layer_norm_bwd_workspace_floats(4, 4, None), "bad argument")
    refused(lib.xdfm_layer_norm_bwd_workspace_floats(4, (1 << 30) + 1, ctypes.byref(size)), "bad argument")
    assert norm_fwd(rows=0, x=None, y=None) == 0  # no rows: nothing to do


def tensor(**kw):
    a = dict(param=1 << 20, grad=2 << 20, slot_m=3 << 20, slot_v=4 << 20, scale_m=None, scale_v=None, n=1000,
             weight_decay=0.0, grad_dtype=0)
    a.update(kw)
    return _lib.AdamWTensor(*[a[k] for k, _ in _lib.AdamWTensor._fields_])


def plan(tensors, bits=32, image=None, size=0):
    table = (_lib.AdamWTensor * max(len(tensors), 1))(*tensors)
    info = _lib.AdamWPlanInfo()
    return lib.xdfm_adamw_plan(table, len(tensors), bits, image, size, ctypes.byref(info)), info


@pytest.mark.parametrize("kw,bits,text", [
    (dict(n=-1), 32, "elements"), (dict(n=1 << 45), 32, "elements"), (dict(grad_dtype=3), 32, "gradient type"),
    (dict(weight_decay=-1.0), 32, "weight_decay"), (dict(weight_decay=float("nan")), 32, "weight_decay"),
    (dict(weight_decay=float("inf")), 32, "weight_decay"), (dict(param=None), 32, "null"), (dict(grad=None), 32, "null"),
    (dict(slot_m=None), 32, "null"), (dict(slot_v=None), 32, "null"), (dict(), 8, "scales"),
    (dict(scale_m=5 << 20), 8, "scales"), (dict(scale_m=5 << 20, scale_v=6 << 20), 32, "no scales"),
    (dict(param=(1 << 20) + 2), 32, "misaligned"), (dict(grad=(2 << 20) + 1, grad_dtype=1), 32, "misaligned"),
    (dict(grad=(2 << 20) + 2), 32, "misaligned"), (dict(slot_v=(4 << 20) + 1), 32, "misaligned"),
    (dict(slot_m=1 << 20), 32, "overlap"), (dict(slot_v=(3 << 20) + 3996), 32, "overlap"),
    (dict(grad=1 << 20), 32, "gradient of tensor 0"), (dict(grad=(1 << 20) - 2000), 32, "gradient of tensor 0"),
    (dict(grad=(4 << 20) + 3996), 32, "gradient of tensor 0"),
    (dict(scale_m=5 << 20, scale_v=(5 << 20) + 15), 8, "overlap"),
])
def test_adamw_plan_refuses(kw, bits, text):
    refused(plan([tensor(**kw)], bits)[0], text)


def test_adamw_plan_takes_neighbours_and_refuses_the_same_tensor_twice():
    a = tensor()
    b = tensor(param=(1 << 20) + 4000, grad=(2 << 20) + 4000, slot_m=(3 << 20) + 4000, slot_v=(4 << 20) + 4000)
    rc, info = plan([a, b])
    assert rc == 0 and info.elements == 2000 and info.chunks == 2 and info.state_bits == 32
    # a shared gradient is only read
    assert plan([a, tensor(param=(1 << 20) + 4000, slot_m=(3 << 20) + 4000, slot_v=(4 << 20) + 4000)])[0] == 0
    refused(plan([a, a])[0], "overlap")
    refused(plan([a], 16)[0], "32 or 8 bits")
    refused(lib.xdfm_adamw_plan(None, 1, 32, None, 0, ctypes.byref(info)), "bad argument")
    refused(lib.xdfm_adamw_plan(None, 0, 32, None, 0, None), "bad argument")
    # no tensors, tensors without elements
    assert plan([])[0] == 0 and plan([tensor(n=0, param=None, grad=None)])[1].chunks == 0
    refused(plan([tensor(n=1 << 44)])[0], "too many")


def test_adamw_plan_image():
    t = tensor(n=10000, scale_m=5 << 20, scale_v=6 << 20, grad_dtype=1, weight_decay=0.25)
    rc, info = plan([tensor(n=0), t], 8)
    assert rc == 0
    image = (ctypes.c_int64 * (info.bytes // 8))()
    refused(plan([tensor(n=0), t], 8, ctypes.addressof(image), info.bytes - 8)[0], "bytes", code=-3)
    assert plan([tensor(n=0), t], 8, ctypes.addressof(image), info.bytes)[0] == 0
    size = info.bytes // info.chunks // 8
    records = [list(image[k * size:(k + 1) * size]) for k in range(info.chunks)]
    at = 0
    for r in records:
        count, index = r[8] & 0xFFFFFFFF, r[8] >> 32
        assert r[:8] == [(1 << 20) + 4 * at, (2 << 20) + 2 * at, (3 << 20) + at, (4 << 20) + at, (5 << 20) + at // 64,
                         (6 << 20) + at // 64, at, at]
        assert index == 1 and at % 64 == 0 and 0 < count <= info.chunk_elems
        at += count
    assert at == 10000


def test_adamw_step_refuses():
    _, info = plan([tensor()])
    good = dict(lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, step=1)

    def step(plan_ptr=4096, i=info, **kw):
        a = _lib.AdamWArgs()
        for k, v in dict(good, **kw).items():
            setattr(a, k, v)
        return lib.xdfm_adamw_step(plan_ptr, ctypes.byref(i), ctypes.byref(a), None)

    nan, inf = float("nan"), float("inf")
    for kw, text in ((dict(lr=-1.0), "lr"), (dict(lr=nan), "lr"), (dict(lr=inf), "lr"), (dict(beta1=1.0), "beta1"),
                     (dict(beta1=-0.1), "beta1"), (dict(beta2=1.0), "beta2"), (dict(beta2=nan), "beta2"),
                     (dict(eps=0.0), "eps"), (dict(eps=-1e-8), "eps"), (dict(eps=1e-60), "eps"), (dict(eps=1e-31), "eps"), (dict(eps=inf), "eps"), (dict(eps=nan), "eps"),
                     (dict(step=0), "steps count"), (dict(step=-3), "steps count"), (dict(plan_ptr=None), "null"),
                     (dict(plan_ptr=4100), "misaligned")):
        refused(step(**kw), text)
    refused(lib.xdfm_adamw_step(4096, None, None, None), "null")
    refused(lib.xdfm_adamw_step(4096, ctypes.byref(info), None, None), "null")
    wrong = _lib.AdamWPlanInfo(info.bytes, info.chunks + 1, info.elements, 32, info.chunk_elems)
    refused(step(i=wrong), "not what xdfm_adamw_plan gave")
    refused(step(i=_lib.AdamWPlanInfo()), "not what xdfm_adamw_plan gave")
    refused(lib.xdfm_adamw_state_read(4096, ctypes.byref(info), 64, 64, None), "32-bit states")
    refused(lib.xdfm_adamw_state_write(4096, ctypes.byref(info), 64, 64, None), "32-bit states")
    _, info8 = plan([tensor(scale_m=5 << 20, scale_v=6 << 20)], 8)
    refused(lib.xdfm_adamw_state_read(4096, ctypes.byref(info8), None, 64, None), "null")
    refused(lib.xdfm_adamw_state_read(4096, ctypes.byref(info8), 64, 65, None), "misaligned")
    refused(lib.xdfm_adamw_state_write(4096, ctypes.byref(info8), 64, None, None), "null")
    refused(lib.xdfm_adamw_state_write(4096, ctypes.byref(info8), 66, 64, None), "misaligned")
    # nothing to do
    _, none = plan([])
    assert step(plan_ptr=None, i=none) == 0


def test_the_class_refuses_what_the_library_cannot_see():
    p, g = torch.zeros(8), torch.zeros(8)
    with pytest.raises(ValueError, match="GPU"):
        AdamW([p], [g])
    with pytest.raises(ValueError, match="at least one"):
        AdamW([], [])
    with pytest.raises(ValueError, match="32 or 8"):
        AdamW([p], [g], state_bits=16)
    with pytest.raises(ValueError, match="gradients"):
        AdamW([p], [g, g])
    assert ctypes.sizeof(_lib.AdamWTensor) == 64 and ctypes.sizeof(_lib.AdamWArgs) == 56
    assert ctypes.sizeof(_lib.AdamWPlanInfo) == 32
