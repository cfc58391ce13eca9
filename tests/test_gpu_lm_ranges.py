"""Layer norm, token log probabilities and AdamW at the ends of what they take: rows whose logits rise by powers of ten,
norms of constant rows far from zero, several rows per team of waves, 8-bit states of elements that are small in their block.
Against plain implementations in 64 bits, with the tolerances of test_gpu_lm_operators."""
import numpy as np
import pytest

import lm_reference as ref
from lm_reference import U32, Matrix, Raw
from polarai_framework_amd import capi
from test_gpu_lm_operators import close, logprob_tolerances, norm_tolerances

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


# ---- log probabilities ------------------------------------------------------------

TILE = {"f32": 4096, "f16": 8192, "bf16": 8192}   # logits that a work-group takes at a time
LARGEST = {"f32": float(np.finfo(np.float32).max), "f16": 65504.0, "bf16": float(ref.widen(np.array([0x7F7F], np.uint16), "bf16")[0])}


def check_repeated_rows(dev, patterns, rows, kind, scale):
    """Rows that repeat a few patterns, so that there are many of them (which sets how a row is cut into parts) and few to
    compute in 64 bits."""
    n, cols = patterns.shape
    which = np.arange(rows) % n
    tokens = np.argmax(patterns, 1)
    r = ref.logprob(patterns, tokens, scale)
    X, T = Matrix(dev, kind, rows, cols, cols + 1, 1, patterns[which]), Raw(dev, tokens[which].astype(np.int64))
    LP, H, S = Raw(dev, np.full(rows, 9, np.float32)), Raw(dev, np.full(rows, 9, np.float32)), Raw(dev, np.full((rows, 2), 9, np.float32))
    dev.flogprob(X, T, LP, rows, cols, scale=scale, stats=S, entropy=H, dtype=kind, stride=X.stride)
    logsum_tol, lp_tol, entropy_tol = logprob_tolerances(r)
    stats = S.values()
    assert np.array_equal(stats[:, 0], r["stats"][which, 0])
    close(stats[:, 1], r["stats"][which, 1], logsum_tol[which], "logsum")
    close(H.values(), r["entropy"][which], entropy_tol[which], "entropy")
    close(LP.values(), r["logprob"][which], lp_tol[np.arange(n), tokens][which], "logprob")
    for t in (X, T, LP, H, S):
        t.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,tiles", [(520, 3), (64, 24), (3, 5)])
def test_logprob_of_rows_that_rise_before_one_large_logit(dev, kind, rows, tiles):
    """A wave that has summed terms far above its reference when one very large logit (a forced token) makes all of them
    nothing: the entropy is that of the large one alone, 0."""
    _say("flogprob rise", kind, rows, tiles)
    tile = TILE[kind]
    cols = tiles * tile - 5
    step = np.arange(cols) // tile % 3
    top = min(1e30, LARGEST[kind] / 2)

    def row(first, then, last, at):
        x = np.where(step == 0, first, then).astype(np.float64)
        if last is not None:
            x[at] = last
        return x
    end = 2 * tile + 100
    patterns = np.stack([row(0.0, 20.0, top, end), row(5.0, 25.0, LARGEST[kind], end), row(0.0, 40.0, min(1e20, top), cols - 1),
                         row(0.0, 20.0, 70.0, end), row(0.0, 20.0, None, 0), row(-30.0, 10.0, top, 3), row(-np.inf, 40.0, top, end),
                         row(-LARGEST[kind], 20.0, 1000.0, end)])
    check_repeated_rows(dev, ref.rounded(patterns, kind), rows, kind, 1.0)


@pytest.mark.parametrize("scale", [1.0, 1.3, 1.38, 2.0 ** 20])
def test_logprob_of_large_logits_one_step_apart(dev, scale):
    """Logits so large that neighbours of fp32 lie up to 88 apart in the exponential: terms relative to the smaller one would
    be up to 2^128 each."""
    _say("flogprob neighbours", scale)
    rows, tile = 520, TILE["f32"]
    patterns = []
    for size in (6e8, -6e8, 6e8 / 2.0 ** 20, 1.2e9, 3e5):
        low = np.float32(size)
        high = np.nextafter(low, np.float32(np.inf))
        patterns.append(np.where(np.arange(3 * tile) < tile, float(low), float(high)))
        patterns.append(np.where(np.arange(3 * tile) < 2 * tile, float(low), float(high)))
    check_repeated_rows(dev, np.stack(patterns), rows, "f32", scale)


# ---- layer norm -------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 5, 127, 515, 1021, 2500, 5000, 8191, 9001, 33001])
@pytest.mark.parametrize("given", [True, False])
def test_layernorm_grad_of_constant_rows_far_from_zero(dev, kind, cols, given):
    """A constant row has h = 0 everywhere, however large its value: what stands behind the row's end takes no part."""
    _say("flayernorm_grad constant rows", kind, cols, given)
    rng = np.random.default_rng(cols)
    x = ref.rounded(rng.standard_normal((4, cols)), kind)
    # a power of two, whose sum over the row and mean are exact where the statistics are computed again; the reciprocal root
    # of eps is 316, so that 2^121 times it passes what fp32 holds
    x[1] = 2.0 ** 121 if given or cols < 100 else 2.0 ** 112
    x[2] = -2.0 ** 120 if given or cols < 100 else -2.0 ** 111
    eps = 1e-5 if given or cols < 100 else 1e-20
    dy = ref.rounded(rng.standard_normal((4, cols)), kind)
    W = Raw(dev, np.ones(cols, np.float32))
    mean, rstd = x.mean(1), 1 / np.sqrt(x.var(1) + eps)
    DY, X, DX = Matrix(dev, kind, 4, cols, values=dy), Matrix(dev, kind, 4, cols, values=x), Matrix(dev, kind, 4, cols)
    M, R = Raw(dev, mean.astype(np.float32)), Raw(dev, rstd.astype(np.float32))
    DB = Raw(dev, np.zeros(cols, np.float32))
    dev.flayernorm_grad(DY, X, W, DX, None, DB, 4, cols, eps=eps, mean=M if given else None, rstd=R if given else None, dtype=kind)
    got = DX.values()
    for r in (1, 2):
        want = rstd[r] * (dy[r] - dy[r].mean())   # h is 0
        # h is exactly 0 where the mean is exact: it is for rows up to 2^24 elements of one power of two (sums of at most
        # 24 bits of it); the sum along the row as in check_norm_grad, rstd rounded or computed again (8 u)
        tol = rstd[r] * (4 * U32 * (np.abs(dy[r]) + np.abs(dy[r]).mean()) + 64 * U32 * np.abs(dy[r]).mean()) + 10 * U32 * np.abs(want)
        close(got[r], want, tol * 1.01 + ref.HALF_STEP[kind] * np.abs(want) + ref.TINY[kind], f"dx of row {r}")
    assert np.isfinite(got).all()
    close(DB.values(), dy.sum(0), 8 * U32 * np.abs(dy).sum(0), "dbias")
    for t in (W, DY, X, DX, M, R, DB):
        t.free()


@pytest.mark.parametrize("rows,cols,kind", [(13000, 40, "f32"), (13000, 513, "bf16"), (12600, 300, "f32"), (6200, 1500, "f16"), (6200, 700, "f32"),
                                            (2100, 4000, "bf16"), (2100, 2000, "f32"), (1300, 8192, "bf16"), (1300, 4000, "f32"),
                                            (600, 16384, "bf16"), (600, 8000, "f32"), (600, 16384, "f32")])
def test_layernorm_of_several_rows_per_team(dev, rows, cols, kind):
    """More rows than the grid has teams and each of them rows ahead: the registers of the rows that come next are filled
    again and the walk ends inside a round."""
    _say("flayernorm rows per team", rows, cols, kind)
    rng = np.random.default_rng(rows + cols)
    x = ref.rounded(rng.standard_normal((rows, cols)) * 1.5 + rng.standard_normal((rows, 1)) * 3, kind)
    w, b = ref.rounded(1 + 0.3 * rng.standard_normal(cols), "f32"), ref.rounded(0.5 * rng.standard_normal(cols), "f32")
    y, mean, rstd = ref.layernorm(x, w, b, 1e-5)
    X, Y = Matrix(dev, kind, rows, cols, cols + 3, 1, x), Matrix(dev, kind, rows, cols, cols + 1, 2)
    W, B = Raw(dev, w.astype(np.float32)), Raw(dev, b.astype(np.float32))
    M, R = Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros(rows, np.float32))
    dev.flayernorm(X, W, B, Y, rows, cols, mean=M, rstd=R, dtype=kind, x_stride=X.stride, out_stride=Y.stride)
    y_tol, mean_tol, rstd_tol = norm_tolerances(x, w, b, y, mean, rstd, kind)
    close(Y.values(), y, y_tol, "y")
    close(M.values(), mean, mean_tol, "mean")
    close(R.values(), rstd, rstd_tol, "rstd")
    for t in (X, Y, W, B, M, R):
        t.free()


def norm_error_bounds(x, w, mean, rstd, given):
    """(mean_tol, rstd_rel) as in test_gpu_lm_operators: none where the statistics are given."""
    if given:
        return np.zeros((len(x), 1)), np.zeros((len(x), 1))
    mean_tol = 64 * U32 * np.abs(x).mean(1)
    return mean_tol[:, None], (64 * U32 + 0.5 * (rstd * mean_tol) ** 2)[:, None]


def check_norm_grad(dev, x, dy, w, kind, params, given, eps=1e-3):
    rows, cols = x.shape
    _, mean, rstd = ref.layernorm(x, w, 0.0, eps)
    mean32, rstd32 = mean.astype(np.float32), rstd.astype(np.float32)
    mean_, rstd_ = (mean32.astype(np.float64), rstd32.astype(np.float64)) if given else (mean, rstd)
    dx, dw, db = ref.layernorm_grad(dy, x, w, mean_, rstd_)
    mean_tol, rstd_rel = norm_error_bounds(x, w, mean, rstd, given)
    h = np.abs(x - mean_[:, None]) * rstd_[:, None]
    h_tol = rstd_[:, None] * mean_tol + h * (rstd_rel + 3 * U32) + rstd_[:, None] * 2 * U32 * np.abs(mean_[:, None])
    g = np.abs(dy * w)
    along1, alongh = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    alongh_tol = (g * h_tol).mean(1, keepdims=True) + 64 * U32 * alongh
    dx_tol = rstd_[:, None] * (4 * U32 * (g + along1 + h * alongh) + 64 * U32 * along1 + h * alongh_tol + h_tol * alongh)
    dx_tol = dx_tol + np.abs(dx) * (rstd_rel + 2 * U32)
    adds = 32 + rows
    dw_tol = adds * U32 * (np.abs(dy) * h).sum(0) + (np.abs(dy) * h_tol).sum(0)
    db_tol = adds * U32 * np.abs(dy).sum(0)
    DY, X = Matrix(dev, kind, rows, cols, cols + 2, 3, dy), Matrix(dev, kind, rows, cols, cols + 5, 2, x)
    W, M, R = Raw(dev, ref.store(w, params)), Raw(dev, mean32), Raw(dev, rstd32)
    DX = Matrix(dev, kind, rows, cols, cols + 1, 7)
    DW, DB = (Raw(dev, np.zeros(cols, ref.STORED[params])) for _ in range(2))
    dev.flayernorm_grad(DY, X, W, DX, DW, DB, rows, cols, eps=eps, mean=M if given else None, rstd=R if given else None, dtype=kind,
                        param_dtype=params, grad_stride=DY.stride, x_stride=X.stride, dx_stride=DX.stride)
    half = ref.HALF_STEP

    def stored(want, k):
        return half[k] * np.abs(want) + ref.TINY[k]
    close(DX.values(), dx, dx_tol * (1 + half[kind]) + stored(dx, kind), "dx")
    close(ref.widen(DW.values(), params), dw, dw_tol * 1.01 + stored(dw, params), "dweight")
    close(ref.widen(DB.values(), params), db, db_tol * 1.01 + stored(db, params), "dbias")
    for t in (DY, X, W, M, R, DX, DW, DB):
        t.free()


@pytest.mark.parametrize("rows,cols,kind", [(8300, 40, "f32"), (8300, 600, "bf16"), (8300, 300, "f32"), (1600, 2000, "f16"), (1600, 1000, "f32"),
                                            (1300, 4096, "bf16"), (1300, 2048, "f32"), (800, 8192, "bf16"), (800, 4000, "f32"),
                                            (600, 16384, "bf16"), (600, 8192, "f32"), (600, 16384, "f32"), (100, 33000, "bf16"), (100, 33000, "f32")])
@pytest.mark.parametrize("given", [True, False])
def test_layernorm_grad_of_several_rows_per_team(dev, rows, cols, kind, given):
    """As above; every team adds several rows to its columns' sums, in registers and in LDS, and a slice of long rows has
    several of them."""
    _say("flayernorm_grad rows per team", rows, cols, kind, given)
    rng = np.random.default_rng(rows + cols + 1)
    x = ref.rounded(rng.standard_normal((rows, cols)) * 1.5 + rng.standard_normal((rows, 1)) * 3, kind)
    w = ref.rounded(1 + 0.3 * rng.standard_normal(cols), "f32")
    check_norm_grad(dev, x, ref.rounded(rng.standard_normal((rows, cols)), kind), w, kind, "f32", given)


@pytest.mark.parametrize("params", ["f32", "bf16"])
def test_layernorm_grad_over_no_rows_asks_for_no_strides(dev, params):
    _say("flayernorm_grad no rows, no strides")
    DW, DB = (Raw(dev, np.ones(70, ref.STORED[params])) for _ in range(2))
    dev.flayernorm_grad(None, None, None, None, DW, DB, 0, 70, dtype=params, param_dtype=params, grad_stride=0, x_stride=0)
    assert not DW.values().any() and not DB.values().any()
    DW.free(), DB.free()


# ---- AdamW ------------------------------------------------------------------------

def test_adamw_8_bit_states_with_seven_decades_in_a_block(dev):
    """Elements whose gradients are 10 to 10 million times smaller than the largest of their block, down to where neither state
    has a code of its own: their steps stay of the size that AdamW's steps have, a few lr.  What bounds them: |m| / sqrt(v) of
    the unrounded states is about 1 for such gradients (with the corrections 1.1 at most over these steps); a state near the
    smallest code is off by a factor of two at most, m up and the root down, so 4.4; and where the root is below the smallest
    code, m may be a whole code too much, over a divisor of a code: the ratio of the block's two scales, at most 1.1 of its
    corrections.  6 covers the sum."""
    _say("fadamw decades")
    n, steps, lr = 8 * 256, 400, 1e-3
    rng = np.random.default_rng(31)
    decade = np.arange(n) % 8
    decade[(decade == 0) & (np.arange(n) % 256 != 0)] = 1   # the largest is alone in its block
    P, G = Raw(dev, np.zeros(n, np.float32)), Raw(dev, np.zeros(n, np.float32))
    M, V = Raw(dev, np.zeros(n, np.uint8)), Raw(dev, np.zeros(n, np.uint8))
    MS, VS = Raw(dev, np.zeros(n // 256, np.float32)), Raw(dev, np.zeros(n // 256, np.float32))
    plan = capi.adamw_tensors([dict(count=n, param=P, grad=G, m=M, v=V, m_scale=MS, v_scale=VS)])
    before, moved = np.zeros(n), []
    for step in range(1, steps + 1):
        g = (rng.standard_normal(n) * 10.0 ** -decade).astype(np.float32)
        dev.copy_to_device(G.ptr, g.ctypes.data, g.nbytes)
        dev.fadamw(plan, step=step, lr=lr, seed=step, state_dtype="8bit")
        after = P.values().astype(np.float64)
        moved.append((after - before) / lr)
        before = after
    moved = np.array(moved)
    largest = np.abs(moved[10:]).max(0)
    rms = [np.sqrt((moved[10:, decade == d] ** 2).mean()) for d in range(8)]
    for d in range(8):
        _say(f"size 1e-{d}: root mean square {rms[d]:.3f} lr, largest {largest[decade == d].max():.2f} lr")
    assert largest.max() <= 6, largest.max()
    # what has codes of its own moves as with states in 32 bits
    assert all(0.15 < rms[d] < 0.35 for d in (1, 2, 3, 4))
    for t in (P, G, M, V, MS, VS):
        t.free()


def test_adamw_8_bit_roots_below_the_smallest_code(dev):
    """A root that is not zero and rounds to zero leaves its trace: code 0x80, which stands for 0 too; the next step divides by
    the smallest code at least.  A root that is zero leaves code 0."""
    _say("fadamw traces")
    n = 256
    g = np.zeros(n, np.float32)
    g[0], g[1:100], g[100:200] = 1.0, 1e-9, 1e-3
    P, G = Raw(dev, np.zeros(n, np.float32)), Raw(dev, g)
    M, V, MS, VS = Raw(dev, np.zeros(n, np.uint8)), Raw(dev, np.zeros(n, np.uint8)), Raw(dev, np.zeros(1, np.float32)), Raw(dev, np.zeros(1, np.float32))
    plan = capi.adamw_tensors([dict(count=n, param=P, grad=G, m=M, v=V, m_scale=MS, v_scale=VS)])
    dev.fadamw(plan, step=1, lr=1e-3, seed=5, state_dtype="8bit")
    codes = V.values()
    assert (codes[1:100] == 0x80).all() and (codes[200:] == 0).all()
    assert (codes[100:200] > 0).all() and (codes[100:200] < 0x80).all() and codes[0] == 0x7E
    # the states of the 2nd step as given: m one code, the root's trace; gradient 0
    m = np.full(n, 1, np.uint8)
    dev.copy_to_device(M.ptr, m.ctypes.data, n)
    before = P.values().astype(np.float64)
    zero = np.zeros(n, np.float32)
    dev.copy_to_device(G.ptr, zero.ctypes.data, zero.nbytes)
    ms, vs = float(MS.values()[0]), float(VS.values()[0])
    dev.fadamw(plan, step=2, lr=1e-3, seed=6, state_dtype="8bit", eps=0.0)
    step = before - P.values()
    m2 = 0.9 * 2.0 ** -9 * ms / (1 - 0.9 ** 2)
    want = 1e-3 * m2 / (2.0 ** -9 * vs / np.sqrt(1 - 0.999 ** 2))
    # about ten roundings and a reciprocal good to 2 u, the difference of parameters of 1e-3
    assert np.abs(step[1:100] - want).max() <= 20 * U32 * want + 4 * U32 * np.abs(before[1:100]).max()
    for t in (P, G, M, V, MS, VS):
        t.free()


def test_adamw_8_bit_lists_over_launches_and_far_element_numbers(dev):
    """More tensors than a launch takes, whose elements' numbers in the random sequence lie beyond 2^32, and for one of them on
    both sides of it: each state within the neighbours that its own random bits allow."""
    _say("fadamw numbers")
    rng = np.random.default_rng(55)
    sizes = [1, 255, 256, 257, 1023, 4097, 7] * 15
    firsts = [[0, (1 << 32) - 100, (1 << 32) + 5, (1 << 40) + 123, (1 << 63) + 1][i % 5] for i in range(len(sizes))]
    made, fields = [], []
    for n, first in zip(sizes, firsts):
        g, p = (rng.standard_normal(n) * 0.1).astype(np.float32), rng.standard_normal(n).astype(np.float32)
        blocks = -(-n // 256)
        t = dict(n=n, first=first, g=g, G=Raw(dev, g), P=Raw(dev, p), M=Raw(dev, np.zeros(n, np.uint8)), V=Raw(dev, np.zeros(n, np.uint8)),
                 MS=Raw(dev, np.zeros(blocks, np.float32)), VS=Raw(dev, np.zeros(blocks, np.float32)))
        made.append(t)
        fields.append(dict(count=n, first=first, param=t["P"], grad=t["G"], m=t["M"], v=t["V"], m_scale=t["MS"], v_scale=t["VS"]))
    dev.fadamw(capi.adamw_tensors(fields), step=1, lr=1e-3, seed=99, state_dtype="8bit")
    for t in made:
        n, wide = t["n"], t["g"].astype(np.float64)
        number = (np.uint64(t["first"]) + np.arange(n, dtype=np.uint64))
        bits = ref.random_bits(99, number)
        for codes, scales, new, random in ((t["M"], t["MS"], 0.1 * wide, bits & np.uint64(0xFFFF)),
                                           (t["V"], t["VS"], np.sqrt(0.001) * np.abs(wide), bits >> np.uint64(16))):
            by = np.arange(n) // 256
            scale = scales.values().astype(np.float64)
            close(scale, ref.block_largest(new) / 448, 8 * U32 * ref.block_largest(new) / 448, "scale")
            at, unit = ref.held_in_8_bits(new, scale[by], random.astype(np.float64))
            near = 10 * U32 * np.abs(new) / scale[by] / unit + 2.0 ** -20
            low, high = np.floor(at - near) * unit, np.floor(at + near) * unit
            got = np.abs(ref.E4M3[codes.values()])
            assert ((got >= np.minimum(low, 448)) & (got <= np.minimum(high, 448))).all(), (n, t["first"])
        for k in ("G", "P", "M", "V", "MS", "VS"):
            t[k].free()


# ---- tensors of another library ---------------------------------------------------

def test_tensors_of_another_library(dev):
    """Device and pinned host memory of torch; what is too short for its type or lies in ordinary host memory is refused before
    a kernel sees it."""
    torch = pytest.importorskip("torch")
    _say("torch tensors")
    rng = np.random.default_rng(2)
    rows, cols = 5, 300
    x = ref.rounded(rng.standard_normal((rows, cols)), "bf16")
    X = torch.tensor(x, dtype=torch.bfloat16, device="cuda")
    Y = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    W = torch.ones(cols).pin_memory()
    torch.cuda.synchronize()
    dev.flayernorm(X, W, None, Y, rows, cols, dtype="bf16")
    dev.synchronize()
    y, mean, rstd = ref.layernorm(x, np.ones(cols), 0.0, 1e-5)
    close(Y.double().cpu().numpy(), y, norm_tolerances(x, np.ones(cols), np.zeros(cols), y, mean, rstd, "bf16")[0], "y")
    with pytest.raises(ValueError, match="x holds 3000 bytes, 6000"):
        dev.flayernorm(X, None, None, torch.empty(rows, cols, device="cuda"), rows, cols)
    with pytest.raises(TypeError, match="weight"):
        dev.flayernorm(X, torch.ones(cols), None, Y, rows, cols, dtype="bf16")
    with pytest.raises(ValueError, match="tokens"):
        dev.flogprob(X, torch.zeros(rows, dtype=torch.int32, device="cuda"), Y, rows, cols, dtype="bf16")
    p, g, m, v = (torch.full((100,), c, device="cuda") for c in (1.0, 0.5, 0.0, 0.0))
    torch.cuda.synchronize()
    plan = capi.adamw_tensors([dict(count=100, param=p, grad=g, m=m, v=v)])
    with pytest.raises(ValueError, match="grad"):
        dev.fadamw(capi.adamw_tensors([dict(count=100, param=p, grad=g.bfloat16(), m=m, v=v)]), step=1, lr=1e-3)
    dev.fadamw(plan, step=1, lr=1e-3)
    dev.synchronize()
    assert np.abs(p.cpu().numpy() - (1 - 1e-3)).max() <= 4 * U32
