"""What xdfm_adamw_plan and xdfm_adamw_step refuse beyond single arguments: calls whose tensors, sizes or numbers the step
cannot hold (runs without a GPU)."""
import ctypes

import pytest

from recommenders_amd import _lib

lib = _lib.lib


def refused(rc, text, code=-1):
    assert rc == code, rc
    assert text in lib.xdfm_last_error().decode(), lib.xdfm_last_error()


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
    (dict(slot_m=1 << 20), 32, "overlap"), (dict(slot_v=(3 << 20) + 3996), 32, "overlap"),
    (dict(grad=1 << 20), 32, "gradient of tensor 0"), (dict(grad=(4 << 20) + 3996), 32, "gradient of tensor 0"),
    (dict(scale_m=5 << 20, scale_v=(5 << 20) + 15), 8, "overlap"),
])
def test_overlaps_are_refused_where_the_image_is_written_too(kw, bits, text):
    """A caller that knows the image's size from tensors of the same sizes makes the second call alone."""
    apart = dict(scale_m=5 << 20, scale_v=6 << 20) if bits == 8 else {}
    rc, info = plan([tensor(**apart)], bits)
    assert rc == 0
    image = (ctypes.c_int64 * (info.bytes // 8))(*[7] * (info.bytes // 8))
    refused(plan([tensor(**kw)], bits, ctypes.addressof(image), info.bytes)[0], text)
    assert list(image) == [7] * (info.bytes // 8)
    assert plan([tensor(**apart)], bits, ctypes.addressof(image), info.bytes)[0] == 0
    assert list(image)[0] == 1 << 20
