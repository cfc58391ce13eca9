"""CPU tests of the language-model operators: what the entry points refuse
(before they touch a device), and the gradients' formulas against differences
of the forward pass, in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import lm_reference as ref
from polarai_framework_amd import capi

INVALID = 1
A = 1 << 20  # an address that a refused call never looks at


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


@pytest.fixture(scope="module")
def handle():
    """Stands for an opened device: every refusal comes before its first use."""
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


def refused(lib, status, *words):
    assert status == INVALID
    message = lib.polar_hip_last_error().decode()
    for w in words:
        assert w in message, message


NORM = dict(dev=None, type=0, x=A, xStride=8, paramType=0, weight=A, bias=A, eps=1e-5, y=A + 4096, yStride=8, mean=A, rstd=A,
            rows=4, cols=8)
NORM_GRAD = dict(dev=None, type=0, dy=A, dyStride=8, x=A, xStride=8, paramType=0, weight=A, mean=A, rstd=A, eps=1e-5, dx=A + 4096,
                 dxStride=8, dweight=A, dbias=A, rows=4, cols=8)
LOGPROB = dict(dev=None, type=0, logits=A, stride=8, tokenType=1, tokens=A, scale=1.0, logprob=A, stats=A, entropy=A, top=2,
               topIndex=A, topLogprob=A, rows=4, cols=8)
LOGPROB_GRAD = dict(dev=None, type=0, logits=A, stride=8, tokenType=1, tokens=A, scale=1.0, stats=A, dlogprob=A, entropy=A,
                    dentropy=A, dlogits=A + 4096, dlogitsStride=8, rows=4, cols=8)


@pytest.mark.parametrize("change,words", [
    (dict(dev=0), "dev is null"), (dict(type=3), "element type"), (dict(type=-1), "element type"),
    (dict(paramType=1), "parameters"), (dict(type=1, paramType=2), "parameters"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(cols=0), "rows of 1"),
    (dict(cols=(1 << 24) + 1, xStride=1 << 25, yStride=1 << 25), "rows of 1"), (dict(x=0), "null"), (dict(y=0), "null"),
    (dict(xStride=7), "stride"), (dict(yStride=7), "stride"), (dict(rows=1 << 60, xStride=1 << 20), "too large"),
    (dict(x=A + 1), "misaligned"), (dict(y=A + 2), "misaligned"), (dict(weight=A + 2), "misaligned"),
    (dict(mean=A + 2), "misaligned"), (dict(y=A, yStride=9), "in place")])
def test_layernorm_refuses(lib, handle, change, words):
    call = {**NORM, "dev": handle, **change}
    refused(lib, lib.polar_hip_flayernorm(*call.values()), "polar_hip_flayernorm", words)


@pytest.mark.parametrize("change,words", [
    (dict(dev=0), "dev is null"), (dict(type=7), "element type"), (dict(paramType=2), "parameters"),
    (dict(mean=0), "together"), (dict(rstd=0), "together"), (dict(mean=0, rstd=0, eps=-1e-9), "eps"), (dict(cols=0), "rows of 1"),
    (dict(rows=1 << 31), "too many rows"), (dict(dy=0), "null"), (dict(x=0), "null"), (dict(dyStride=7), "stride"),
    (dict(xStride=1), "stride"), (dict(dxStride=7), "stride"), (dict(dx=A, dxStride=9), "in place"),
    (dict(dbias=A + 1), "misaligned")])
def test_layernorm_grad_refuses(lib, handle, change, words):
    call = {**NORM_GRAD, "dev": handle, **change}
    refused(lib, lib.polar_hip_flayernorm_grad(*call.values()), "polar_hip_flayernorm_grad", words)


@pytest.mark.parametrize("change,words", [
    (dict(dev=0), "dev is null"), (dict(type=3), "element type"), (dict(tokenType=3), "token type"), (dict(cols=0), "rows of 1"),
    (dict(cols=(1 << 24) + 1, stride=1 << 25), "rows of 1"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=4e19), "scale"), (dict(scale=1e-20), "scale"), (dict(top=33, cols=100, stride=100), "alternatives"),
    (dict(top=9), "alternatives"), (dict(logits=0), "null"), (dict(tokens=0), "tokens"), (dict(topIndex=0), "alternatives"),
    (dict(topLogprob=0), "alternatives"), (dict(stride=7), "stride"), (dict(tokens=A + 4), "misaligned"),
    (dict(logits=A + 2), "misaligned"), (dict(rows=1 << 62), "too large")])
def test_logprob_refuses(lib, handle, change, words):
    call = {**LOGPROB, "dev": handle, **change}
    refused(lib, lib.polar_hip_flogprob(*call.values()), "polar_hip_flogprob", words)


@pytest.mark.parametrize("change,words", [
    (dict(dev=0), "dev is null"), (dict(type=3), "element type"), (dict(tokenType=-1), "token type"), (dict(cols=0), "rows of 1"),
    (dict(scale=0.0), "scale"), (dict(dlogits=0), "null"), (dict(logits=0), "null"),
    (dict(tokens=0), "tokens"), (dict(entropy=0), "entropy"), (dict(stride=7), "stride"), (dict(dlogitsStride=7), "stride"),
    (dict(dlogits=A, dlogitsStride=9), "in place"), (dict(dlogits=A + 1), "misaligned")])
def test_logprob_grad_refuses(lib, handle, change, words):
    call = {**LOGPROB_GRAD, "dev": handle, **change}
    refused(lib, lib.polar_hip_flogprob_grad(*call.values()), "polar_hip_flogprob_grad", words)


TENSOR = dict(count=10, first=0, weight_decay=0.0, param=A, grad=A, m=A, v=A, master=A, m_scale=A, v_scale=A)
CONFIG = dict(param_type=0, grad_type=0, state_bits=32, seed=1, step=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0)


@pytest.mark.parametrize("config,tensor,words", [
    (dict(param_type=3), {}, "element type"), (dict(grad_type=-1), {}, "element type"), (dict(state_bits=16), {}, "32 or 8"),
    (dict(step=0), {}, "from 1"), (dict(beta1=1.0), {}, "beta1"), (dict(beta2=-0.1), {}, "beta1"),
    (dict(beta2=float("nan")), {}, "beta1"), (dict(lr=float("inf")), {}, "finite"), (dict(eps=-1.0), {}, "finite"),
    (dict(grad_scale=float("nan")), {}, "finite"), ({}, dict(param=0), "null"), ({}, dict(grad=0), "null"), ({}, dict(m=0), "null"),
    ({}, dict(v=0), "null"), (dict(param_type=2), dict(master=0), "master"), (dict(state_bits=8), dict(m_scale=0), "scales"),
    (dict(state_bits=8), dict(v_scale=0), "scales"), ({}, dict(count=(1 << 33) + 1), "too large"),
    ({}, dict(weight_decay=float("nan")), "decay"), ({}, dict(m=A + 1), "misaligned"), ({}, dict(param=A + 2), "misaligned")])
def test_adamw_refuses(lib, handle, config, tensor, words):
    # the second tensor of the list is the wrong one: nothing is launched for the first either
    tensors = capi.adamw_tensors([{**TENSOR, "param": A + 4096}, {**TENSOR, **tensor}])
    c = capi.AdamWConfig(*{**CONFIG, **config}.values())
    refused(lib, lib.polar_hip_fadamw(handle, C.byref(c), tensors, 2), "polar_hip_fadamw", words)


def test_adamw_refuses_parameters_that_overlap(lib, handle):
    c = capi.AdamWConfig(*CONFIG.values())
    for at in (A, A + 36, A - 36):   # ten elements of four bytes each
        tensors = capi.adamw_tensors([TENSOR, {**TENSOR, "param": A + 8192}, {**TENSOR, "param": at}])
        refused(lib, lib.polar_hip_fadamw(handle, C.byref(c), tensors, 3), "overlap")


def test_adamw_refuses_null_arguments(lib, handle):
    c = capi.AdamWConfig(*CONFIG.values())
    refused(lib, lib.polar_hip_fadamw(None, C.byref(c), None, 0), "null")
    refused(lib, lib.polar_hip_fadamw(handle, None, None, 0), "null")
    refused(lib, lib.polar_hip_fadamw(handle, C.byref(c), None, 1), "null list")
    with pytest.raises(KeyError):
        capi.adamw_tensors([dict(weights=A)])


def test_no_rows_touch_nothing(lib, handle):
    """Null tensors are fine where there are no rows, and nothing is asked of the device."""
    assert lib.polar_hip_flayernorm(*{**NORM, "dev": handle, "rows": 0, "x": 0, "y": 0}.values()) == 0
    assert lib.polar_hip_flogprob(*{**LOGPROB, "dev": handle, "rows": 0, "logits": 0}.values()) == 0
    assert lib.polar_hip_flogprob_grad(*{**LOGPROB_GRAD, "dev": handle, "rows": 0, "logits": 0}.values()) == 0
    # no output is asked for
    assert lib.polar_hip_flogprob(*{**LOGPROB, "dev": handle, "logprob": 0, "stats": 0, "entropy": 0, "top": 0}.values()) == 0
    assert lib.polar_hip_flayernorm_grad(*{**NORM_GRAD, "dev": handle, "dx": 0, "dweight": 0, "dbias": 0}.values()) == 0


def differences(f, x, step):
    """Central differences of a scalar function, one element at a time."""
    d = np.empty_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + step
        up = f()
        x[i] = keep - step
        d[i] = (up - f()) / (2 * step)
        x[i] = keep
    return d


def test_layernorm_gradient_formula_against_differences():
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((3, 7)) * 2 + 1, rng.standard_normal((3, 7))
    w, b = 1 + 0.3 * rng.standard_normal(7), rng.standard_normal(7)
    _, mean, rstd = ref.layernorm(x, w, b, 1e-5)
    dx, dw, db = ref.layernorm_grad(dy, x, w, mean, rstd)

    def value():
        return (ref.layernorm(x, w, b, 1e-5)[0] * dy).sum()
    # truncation ~ step^2 times a third derivative of order 10, cancellation ~ 2^-53 * 10 / step: both below 1e-9
    for got, of in ((dx, x), (dw, w), (db, b)):
        assert np.allclose(got, differences(value, of, 1e-6), rtol=0, atol=1e-8)


def test_logprob_gradient_formula_against_differences():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 9)) * 2
    tokens, g, h = np.array([3, -1, 0, 8]), rng.standard_normal(4), rng.standard_normal(4)
    r = ref.logprob(x, tokens, 1.3)
    d, _ = ref.logprob_grad(x, tokens, 1.3, g, h, r)

    def value():
        q = ref.logprob(x, tokens, 1.3)
        return (q["logprob"] * g + q["entropy"] * h).sum()
    assert np.allclose(d, differences(value, x, 1e-6), rtol=0, atol=1e-8)


def test_8_bit_floats_of_the_reference():
    assert ref.E4M3[0x7E] == 448 and ref.E4M3[0x08] == 2.0 ** -6 and ref.E4M3[1] == 2.0 ** -9 and ref.E4M3[0xB8] == -1.0
    assert np.all(np.diff(ref.E4M3[:0x7F]) > 0)


def test_token_head_graphs_call_sequence_on_the_mock_device():
    """Forward, gradient and update graphs of a model head: each launch reaches the device with the operands in order."""
    from polarai_framework_amd import graphs, harness
    x, norm, w = np.ones((3, 4)), np.ones((2, 4)), np.ones((4, 5))
    f, g, u, named = graphs.token_head_graphs(x, norm, w, np.array([1, -1, 4]))
    assert [n.kernel for n in f.nodes if n.kind == "op"] == ["flayernorm", "fmatmul_f_f", "flogprob"]
    assert [n.kernel for n in g.nodes if n.kind == "op"] == ["flogprob_grad", "fmatmul_t_f", "fmatmul_f_t",
                                                             "flayernorm_grad_params", "flayernorm_grad"]
    seed = [n for n in g.nodes if n.name == "seed"][0]
    assert seed.shape == (3,) and np.all(seed.data == np.float32(-0.5))
    assert named["gN"].shape == (2, 4) and named["gW"].shape == (4, 5) and named["gX"].shape == (3, 4)
    with harness.Harness(plugin=None) as h:
        tensors = {}
        for gr in (f, g, u):
            graphs.emit(gr, h, tensors)
            h.run()
            h.clear_program()
        assert h.counters().launches == 3 + 5 + 4


def test_operands_are_buffers_tensors_of_other_libraries_or_addresses():
    class Foreign:
        def data_ptr(self):
            return 4096

    class Own:
        ptr = 8192
    plan = capi.adamw_tensors([dict(count=3, param=Foreign(), grad=Own(), m=12288, v=None, weight_decay=0.25, first=1 << 40)])
    assert (plan[0].param, plan[0].grad, plan[0].m, plan[0].v) == (4096, 8192, 12288, None)
    assert (plan[0].count, plan[0].first, plan[0].weight_decay, plan[0].master) == (3, 1 << 40, 0.25, None)
