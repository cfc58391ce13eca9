"""CPU tests of how the language-model operators are called: what is refused because two tensors of AdamW would be written by
two work-groups at once, settings that fp32 does not hold, calls over no rows, and operands of other libraries."""
import ctypes as C
import gc
import weakref

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


# ---- operands of other libraries ------------------------------------------------------

class Foreign:
    """What the binding asks of a tensor of another library."""

    def __init__(self, where=0, nbytes=1 << 20, at=A):
        self.where, self.nbytes, self.at = where, nbytes, at

    def get_device(self):
        return self.where

    def data_ptr(self):
        return self.at


class Recorder(capi.Device):
    """A device whose calls are noted instead of made."""

    def __init__(self, ordinal=0):
        self.calls, self.handle, self.ordinal = [], None, ordinal
        outer = self

        class Lib:
            def __getattr__(self, name):
                return lambda *a: outer.calls.append((name, a)) or 0
        self.lib = Lib()


CALLS = {
    "flayernorm": (["x", "weight", "bias", "out", "mean", "rstd"], dict(rows=4, cols=8)),
    "flayernorm_grad": (["grad", "x", "weight", "dx", "dweight", "dbias", "mean", "rstd"], dict(rows=4, cols=8)),
    "flogprob": (["logits", "tokens", "logprob", "stats", "entropy", "top_index", "top_logprob"], dict(rows=4, cols=8, top=2)),
    "flogprob_grad": (["logits", "tokens", "stats", "dlogprob", "dlogits", "entropy", "dentropy"], dict(rows=4, cols=8)),
}
# bytes that four rows of eight fp32 elements, int64 tokens and two alternatives need
BYTES = dict(x=128, out=128, grad=128, dx=128, logits=128, dlogits=128, weight=32, bias=32, dweight=32, dbias=32, mean=16, rstd=16,
             tokens=32, logprob=16, stats=32, entropy=16, dlogprob=16, dentropy=16, top_index=32, top_logprob=32)


@pytest.mark.parametrize("name,operand", [(n, o) for n, (operands, _) in CALLS.items() for o in operands])
def test_operands_of_other_places_and_sizes_are_refused(name, operand):
    operands, sizes = CALLS[name]
    fine = {o: Foreign(nbytes=BYTES[o]) for o in operands}
    dev = Recorder()
    getattr(dev, name)(**fine, **sizes)
    assert len(dev.calls) == 1
    for wrong in (Foreign(where=-1), Foreign(where=1), Foreign(nbytes=BYTES[operand] - 1)):
        with pytest.raises((TypeError, ValueError)) as e:
            getattr(dev, name)(**{**fine, operand: wrong}, **sizes)
        assert operand in str(e.value)
    assert len(dev.calls) == 1   # none of these was made


def test_tensors_of_the_host_are_refused():
    torch = pytest.importorskip("torch")
    dev = Recorder()
    with pytest.raises(TypeError, match="x"):
        dev.flayernorm(torch.zeros(4, 8), None, None, A, 4, 8)
    with pytest.raises(TypeError, match="tokens"):
        dev.flogprob(A, torch.zeros(4, dtype=torch.int64), A, 4, 8)
    with pytest.raises(TypeError, match="grad"):
        capi.adamw_tensors([dict(count=4, param=A, grad=torch.zeros(4), m=A, v=A)])
    assert not dev.calls


def test_strided_rows_need_no_more_than_their_elements():
    """Rows inside a wider buffer: the tensor that is handed over counts rows x columns; one row needs no stride."""
    dev = Recorder()
    dev.flayernorm(Foreign(nbytes=4 * 8 * 2), None, None, Foreign(nbytes=4 * 8 * 2), 4, 8, dtype="bf16", x_stride=100, out_stride=50)
    dev.flogprob(A, Foreign(nbytes=16), None, 4, 8, stats=A, token_dtype="i32")
    assert len(dev.calls) == 2


def test_adamw_lists_keep_their_tensors():
    """The list is made once and used at every step: what it points to lives as long as it does."""
    made = Foreign(nbytes=12)
    alive = weakref.ref(made)
    plan = capi.adamw_tensors([dict(count=3, param=made, grad=A, m=A, v=A)])
    del made
    gc.collect()
    assert alive() is not None and plan[0].param == A
    del plan
    gc.collect()
    assert alive() is None


def test_adamw_lists_are_checked_against_the_device_and_the_call():
    dev = Recorder()
    config = dict(step=1, lr=1e-3)
    dev.fadamw(capi.adamw_tensors([dict(count=3, param=Foreign(nbytes=12), grad=Foreign(nbytes=12), m=A, v=A)]), **config)
    assert len(dev.calls) == 1
    with pytest.raises(TypeError, match="device"):
        dev.fadamw(capi.adamw_tensors([dict(count=3, param=A, grad=Foreign(where=1), m=A, v=A)]), **config)
    # six bytes are three bf16 elements, but not three fp32 ones
    short = capi.adamw_tensors([dict(count=3, param=A, grad=Foreign(nbytes=6), m=A, v=A, master=A)])
    dev.fadamw(short, grad_dtype="bf16", **config)
    with pytest.raises(ValueError, match="grad"):
        dev.fadamw(short, **config)
    eight = capi.adamw_tensors([dict(count=300, param=A, grad=A, m=Foreign(nbytes=300), v=Foreign(nbytes=300), m_scale=Foreign(nbytes=8),
                                     v_scale=Foreign(nbytes=8))])
    dev.fadamw(eight, state_dtype="8bit", **config)
    with pytest.raises(ValueError, match="m"):
        dev.fadamw(eight, **config)
    with pytest.raises(ValueError, match="m_scale"):
        dev.fadamw(capi.adamw_tensors([dict(count=300, param=A, grad=A, m=A, v=A, m_scale=Foreign(nbytes=4), v_scale=A)]),
                   state_dtype="8bit", **config)
    assert len(dev.calls) == 3


def test_adamw_lists_take_new_gradients():
    """A gradient that moved: its address is put into the list."""
    plan = capi.adamw_tensors([dict(count=3, param=A, grad=A, m=A, v=A)])
    plan[0].grad = A + 64
    dev = Recorder()
    dev.fadamw(plan, step=1, lr=1e-3)
    assert dev.calls[0][1][2][0].grad == A + 64
