"""CPU tests of how the language-model operators are called: what is refused because two tensors of AdamW would be written by
two work-groups at once, settings that fp32 does not hold, calls over no rows, and operands of other libraries."""
import ctypes as C

import pytest

from polarai_framework_amd import capi
from test_lm_operators import A, CONFIG, NORM_GRAD, TENSOR, handle, lib, refused  # noqa: F401  (fixtures)


def tensor(i, **change):
    """Ten elements whose buffers lie apart from those of every other i."""
    at = A + (i << 12)
    return {**TENSOR, "param": at, "grad": at + 256, "m": at + 512, "v": at + 768, "master": at + 1024, "m_scale": at + 1280,
            "v_scale": at + 1536, **change}


def step(lib, handle, tensors, **config):  # noqa: F811
    c = capi.AdamWConfig(*{**CONFIG, **config}.values())
    return lib.polar_hip_fadamw(handle, C.byref(c), capi.adamw_tensors(tensors), len(tensors))


@pytest.mark.parametrize("field", ["param", "m", "v", "master", "m_scale", "v_scale"])
@pytest.mark.parametrize("off", [0, 8, -8])
def test_adamw_refuses_whatever_is_written_twice(lib, handle, field, off):  # noqa: F811
    config = dict(param_type=2, grad_type=2, state_bits=8)
    if field.endswith("scale"):
        off //= 4   # a scale or two per tensor: 257 elements
    elif field in ("m", "v"):
        off //= 2   # ten bytes each
    count = 257 if field.endswith("scale") else 10
    tensors = [tensor(i, count=count) for i in range(0, 8, 2)]
    tensors[2][field] = tensors[0][field] + off // 4 * 4 if field.endswith("scale") else tensors[0][field] + off
    refused(lib, step(lib, handle, tensors, **config), "overlap")


@pytest.mark.parametrize("one,other", [("param", "m"), ("m", "v"), ("v", "param"), ("param", "v")])
def test_adamw_refuses_two_buffers_in_one_place(lib, handle, one, other):  # noqa: F811
    for where in (0, 3):
        tensors = [tensor(i) for i in range(4)]
        tensors[where][one] = tensors[1][other]
        refused(lib, step(lib, handle, tensors), "overlap")
    only = tensor(0)
    only[one] = only[other]
    refused(lib, step(lib, handle, [only]), "overlap")


def test_adamw_refuses_a_master_that_is_the_copy(lib, handle):  # noqa: F811
    only = tensor(0)
    only["master"] = only["param"]
    refused(lib, step(lib, handle, [only], param_type=1), "overlap")


@pytest.mark.parametrize("change", [dict(lr=1e300), dict(lr=1e38, beta1=0.999), dict(grad_scale=-1e39), dict(eps=1e39), dict(eps=1e-46), dict(eps=1e-39, state_bits=8)])
def test_adamw_refuses_settings_that_fp32_does_not_hold(lib, handle, change):  # noqa: F811
    refused(lib, step(lib, handle, [tensor(0)], **change), "fp32")


def test_adamw_refuses_a_decay_that_fp32_does_not_hold(lib, handle):  # noqa: F811
    refused(lib, step(lib, handle, [tensor(0), tensor(1, weight_decay=1e60)]), "decay")


def test_layernorm_grad_over_no_rows_takes_any_strides(lib, handle):  # noqa: F811
    call = {**NORM_GRAD, "dev": handle, "rows": 0, "dx": 0, "dweight": 0, "dbias": 0, "dyStride": 0, "xStride": 3, "dxStride": 0}
    assert lib.polar_hip_flayernorm_grad(*call.values()) == 0
