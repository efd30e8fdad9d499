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


def far(n):
    """A tensor of n elements whose arrays lie 2^44 bytes apart."""
    return tensor(param=1 << 44, grad=2 << 44, slot_m=3 << 44, slot_v=4 << 44, n=n)


def test_a_plan_of_more_chunks_than_a_launch_takes_is_refused():
    """256 threads a chunk, and a launch takes fewer than 2^32 threads: 2^24 - 1 chunks."""
    _, info = plan([far(1)])
    most = ((1 << 24) - 1) * info.chunk_elems
    rc, info = plan([far(most)])
    assert rc == 0 and info.chunks == (1 << 24) - 1 and info.elements == most
    refused(plan([far(most + 1)])[0], "too many")
    # in several tensors too
    half = (1 << 23) * info.chunk_elems
    second = tensor(param=5 << 44, grad=6 << 44, slot_m=7 << 44, slot_v=8 << 44, n=half)
    refused(plan([far(half), second])[0], "too many")
    # and a step does not take such an *info from elsewhere
    more = _lib.AdamWPlanInfo((info.chunks + 1) * (info.bytes // info.chunks), info.chunks + 1, info.elements, 32,
                              info.chunk_elems)
    args = _lib.AdamWArgs(0.1, 0.9, 0.999, 1e-8, None, 1, 0)
    refused(lib.xdfm_adamw_step(4096, ctypes.byref(more), ctypes.byref(args), None), "not what xdfm_adamw_plan gave")


def test_a_rate_beyond_what_32_bits_hold_is_refused():
    """lr / (1 - beta1^t) is formed in 32 bits: infinite, it would make NaN of every parameter whose m is 0."""
    _, info = plan([tensor()])
    for lr in (1e39, 3e38, 1.1e20):
        args = _lib.AdamWArgs(lr, 0.9, 0.999, 1e-8, None, 1, 0)
        refused(lib.xdfm_adamw_step(4096, ctypes.byref(info), ctypes.byref(args), None), "lr has to lie in")
