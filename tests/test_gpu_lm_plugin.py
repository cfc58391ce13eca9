"""The language-model operators through the runtime plugin: a model head's
forward, gradient and weight-changing graphs, every node against 64 bits on the
operands that the device consumed, and the shapes that the plugin refuses."""
import subprocess
import sys

import numpy as np
import pytest

import lm_reference as ref
import parity
from lm_reference import U32
from polarai_framework_amd import LIB_PLUGIN, REPO_ROOT, graphs, harness
from test_gpu_lm_operators import close, logprob_tolerances, norm_tolerances

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


@pytest.fixture(params=["heap_ram", "plugin_ram"])
def h(request):
    hh = harness.Harness(plugin=LIB_PLUGIN, plugin_host_memory=request.param == "plugin_ram")
    yield hh
    hh.close()


@pytest.mark.parametrize("rows,cols,classes", [(1, 1, 1), (5, 33, 7), (64, 256, 1000), (130, 777, 5003)])
def test_token_head_graphs(h, rows, cols, classes):
    _say("token head", rows, cols, classes)
    rng = np.random.default_rng(rows + cols)
    x = parity.normal(rng, (rows, cols))
    norm = np.stack([1 + 0.1 * parity.normal(rng, cols), 0.1 * parity.normal(rng, cols)]).astype(np.float32)
    w = parity.normal(rng, (cols, classes), 1 / np.sqrt(cols))
    tokens = rng.integers(0, classes, rows)
    if rows > 3:
        tokens[2] = -1
    f, g, u, named = graphs.token_head_graphs(x, norm, w, tokens.astype(np.float32))
    tensors = {}
    for gr in (f, g):
        graphs.emit(gr, h, tensors)
        h.run()
        h.clear_program()
    v = {n: h.read(tensors[t.tensor_key]).astype(np.float64) for n, t in named.items()}
    wide = x.astype(np.float64)
    y, mean, rstd = ref.layernorm(wide, norm[0].astype(np.float64), norm[1].astype(np.float64), 1e-5)
    close(v["Y"], y, norm_tolerances(wide, norm[0], norm[1], y, mean, rstd, "f32")[0], "Y")
    r = ref.logprob(v["Z"], tokens, 1.0)
    _, lp_tol, _ = logprob_tolerances(r)
    close(v["L"], r["logprob"], lp_tol[np.arange(rows), np.clip(tokens, 0, classes - 1)], "L")
    counted = max(1, int((tokens >= 0).sum()))
    dz, p = ref.logprob_grad(v["Z"], tokens, 1.0, np.full(rows, -1.0 / counted), np.zeros(rows), r)
    # p's exponent: a few u of its terms, and the sums' 128 u; the seed is rounded to fp32
    rel = U32 * (128 + 6 * np.abs(r["z"]) + 8 * np.abs(r["stats"][:, 1:]) + 8 * r["mean_size"][:, None])
    close(v["gZ"], dz, (p * rel + 4 * U32) / counted, "gZ")
    # the products' own bound is 1e-4 of the norm
    for name, want in (("Z", v["Y"] @ w), ("gW", v["Y"].T @ v["gZ"]), ("gY", v["gZ"] @ w.T.astype(np.float64))):
        assert parity.frobenius_rel_error(v[name], want) <= parity.MATMUL_FRO_REL, name
    gx, gw, gb = ref.layernorm_grad(v["gY"], wide, norm[0].astype(np.float64), mean, rstd)
    # normwise: the statistics are good to 64 u times |x| / deviation, the sums over columns and rows to 64 u and rows u of
    # the sum of the sizes, which is within sqrt(n) of the norm
    for name, want, n in (("gX", gx, cols), ("gN", np.stack([gw, gb]), rows)):
        size = np.linalg.norm(v["gY"]) * max(1.0, rstd.max()) * np.sqrt(n) * 4
        assert np.linalg.norm(v[name] - want) <= (256 + rows) * U32 * size, name
    # weights change in place: W + lr * grad
    graphs.emit(u, h, tensors)
    h.run()
    for name, grad, old in (("W", "gW", w), ("N", "gN", norm)):
        want = v[grad].astype(np.float32) * np.float32(-0.01) + old
        assert np.array_equal(h.read(tensors[named[name].tensor_key]), want), name


REFUSALS = {
    "flayernorm's params": "p = h.input(np.ones((1, 8))); h.end_cluster(); h.node('flayernorm', [x, p, 1e-5, h.tensor(4, 8)], 3)",
    "flayernorm_grad's gradient": "g, p = h.input(np.ones((3, 8))), h.input(np.ones((2, 8))); h.end_cluster(); "
                                  "h.node('flayernorm_grad', [g, x, p, 1e-5, h.tensor(4, 8)], 4)",
    "flogprob's tokens": "t = h.input(np.ones(3)); h.end_cluster(); h.node('flogprob', [x, t, 1.0, h.tensor(4)], 3)",
    "flogprob_grad's result": "t, g = h.input(np.ones(4)), h.input(np.ones(4)); h.end_cluster(); "
                              "h.node('flogprob_grad', [x, t, g, 1.0, h.tensor(4, 7)], 4)",
}


@pytest.mark.parametrize("what", REFUSALS)
def test_wrong_shapes_terminate(what):
    """The framework's convention for a launch that cannot be: a message and the end of the process, before anything is
    enqueued."""
    _say("refusal", what)
    code = f"""
import sys; sys.path.insert(0, {REPO_ROOT!r})
import __graft_entry__ as e; e.load_package()
import numpy as np
from polarai_framework_amd import harness, LIB_PLUGIN
h = harness.Harness(plugin=LIB_PLUGIN)
x = h.input(np.ones((4, 8)))
{REFUSALS[what]}
h.end_cluster()
h.run()
print("ran")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode != 0 and "ran" not in r.stdout
    assert what.split("'")[0] in r.stderr
