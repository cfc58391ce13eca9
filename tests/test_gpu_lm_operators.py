"""Layer norm, token log probabilities and AdamW on the device, against plain
implementations in 64 bits.  Tolerances count roundings: u = 2^-24 is half a
step of fp32, a result stored in fewer bits is off by half a step of its type
at most, and a sum in which a value passes through n additions is off by n u
times the sum of the sizes."""
import math

import numpy as np
import pytest

import lm_reference as ref
from lm_reference import HALF_STEP, TINY, U32, Matrix, Raw
from polarai_framework_amd import capi

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


def close(got, want, tol, what):
    got, want, tol = np.broadcast_arrays(got, want, tol)
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    if not ok.all():
        i = tuple(np.argwhere(~ok)[0])
        raise AssertionError(f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, first at {i}: got {got[i]!r}, "
                             f"want {want[i]!r}, tolerance {tol[i]!r}")


def stored_tolerance(want, kind):
    return HALF_STEP[kind] * np.abs(want) + TINY[kind]


# ---- layer norm -------------------------------------------------------------------
# Additions a value passes through in a row's sum: at most 16 in its lane (rows held
# in registers) or (cols / 8192 + 1) + 8 (longer ones), six in the wave, 16 over the
# waves; with the division and the square root 64 cover it up to 2^17 columns.
SUM = 64

NORM_TYPES = [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]
NORM_SHAPES = [(1, 1), (3, 1), (1, 2), (5, 7), (2, 8), (7, 63), (4, 64), (9, 255), (3, 257), (2, 511), (6, 513), (2, 784),
               (5, 1021), (3, 1025), (4, 2048), (2, 2500), (3, 4096), (2, 4099), (2, 8191), (1, 8200), (2, 12345),
               (1, 16384), (2, 16391), (1, 40003)]


def norm_inputs(rng, rows, cols, kind, params):
    x = ref.rounded(rng.standard_normal((rows, cols)) * 1.5 + rng.standard_normal((rows, 1)) * 3, kind)
    w = ref.rounded(1 + 0.3 * rng.standard_normal(cols), params)
    b = ref.rounded(0.5 * rng.standard_normal(cols), params)
    return x, w, b


def norm_tolerances(x, w, b, y, mean, rstd, kind):
    size = np.abs(x).mean(1)
    mean_tol = SUM * U32 * size
    # the squares are taken around the computed mean: its error enters squared
    rstd_tol = rstd * (SUM * U32 + 0.5 * (rstd * mean_tol) ** 2)
    h = np.abs(x - mean[:, None]) * rstd[:, None]
    h_tol = rstd[:, None] * (mean_tol[:, None] + 2 * U32 * (np.abs(x) + size[:, None])) + h * (rstd_tol / rstd + 2 * U32)[:, None]
    y_tol = np.abs(w) * h_tol + 3 * U32 * (np.abs(w) * h + np.abs(b))
    return y_tol * (1 + HALF_STEP[kind]) + stored_tolerance(y, kind), mean_tol + U32 * np.abs(mean), rstd_tol


@pytest.mark.parametrize("kind,params", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layernorm(dev, rows, cols, kind, params):
    _say("flayernorm", rows, cols, kind, params)
    rng = np.random.default_rng(rows * 1000 + cols)
    x, w, b = norm_inputs(rng, rows, cols, kind, params)
    for stride, offset, with_params in ((cols, 0, True), (cols + 3, 1, True), (cols + 8, 5, False)):
        ww, bb = (w, b) if with_params else (np.ones(cols), np.zeros(cols))
        y, mean, rstd = ref.layernorm(x, ww, bb, 1e-5)
        X = Matrix(dev, kind, rows, cols, stride, offset, x)
        Y = Matrix(dev, kind, rows, cols, stride + 1, offset + 2)
        W, B = (Raw(dev, ref.store(v, params)) for v in (w, b))
        M, R = Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros(rows, np.float32))
        dev.flayernorm(X, W if with_params else None, B if with_params else None, Y, rows, cols, eps=1e-5, mean=M, rstd=R,
                       dtype=kind, param_dtype=params, x_stride=X.stride, out_stride=Y.stride)
        y_tol, mean_tol, rstd_tol = norm_tolerances(x, ww, bb, y, mean, rstd, kind)
        close(Y.values(), y, y_tol, "y")
        close(M.values(), mean, mean_tol, "mean")
        close(R.values(), rstd, rstd_tol, "rstd")
        # in place, without the statistics: the same bits
        first = Y.values()
        dev.flayernorm(X, W if with_params else None, B if with_params else None, X, rows, cols, eps=1e-5, dtype=kind,
                       param_dtype=params, x_stride=X.stride, out_stride=X.stride)
        assert np.array_equal(X.values(), first)
        for t in (X, Y, W, B, M, R):
            t.free()


@pytest.mark.parametrize("kind,params", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(700, 64), (2100, 96), (1500, 1000), (600, 2048), (5, 33000)])
def test_layernorm_grad(dev, rows, cols, kind, params):
    _say("flayernorm_grad", rows, cols, kind, params)
    rng = np.random.default_rng(rows * 1000 + cols + 1)
    x, w, _ = norm_inputs(rng, rows, cols, kind, params)
    dy = ref.rounded(rng.standard_normal((rows, cols)), kind)
    eps = 1e-3
    _, mean, rstd = ref.layernorm(x, w, 0.0, eps)
    mean32, rstd32 = mean.astype(np.float32), rstd.astype(np.float32)
    DY, X = Matrix(dev, kind, rows, cols, cols + 2, 3, dy), Matrix(dev, kind, rows, cols, cols + 5, 2, x)
    W = Raw(dev, ref.store(w, params))
    M, R = Raw(dev, mean32), Raw(dev, rstd32)
    for given in (True, False):
        if given:
            mean_, rstd_ = mean32.astype(np.float64), rstd32.astype(np.float64)
            mean_tol = rstd_rel = 0.0
        else:
            mean_, rstd_ = mean, rstd
            _, mean_tol, rstd_tol = norm_tolerances(x, w, np.zeros(cols), x, mean, rstd, kind)
            mean_tol, rstd_rel = mean_tol[:, None], (rstd_tol / rstd)[:, None]
        dx, dw, db = ref.layernorm_grad(dy, x, w, mean_, rstd_)
        h = np.abs(x - mean_[:, None]) * rstd_[:, None]
        h_tol = rstd_[:, None] * mean_tol + h * (rstd_rel + 3 * U32) + rstd_[:, None] * 2 * U32 * np.abs(mean_[:, None])
        g = np.abs(dy * w)
        along1, alongh = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
        alongh_tol = (g * h_tol).mean(1, keepdims=True) + SUM * U32 * alongh
        dx_tol = rstd_[:, None] * (4 * U32 * (g + along1 + h * alongh) + SUM * U32 * along1 + h * alongh_tol + h_tol * alongh)
        dx_tol = dx_tol + np.abs(dx) * (rstd_rel + 2 * U32)
        # a column's sum: rows of a team one after the other, then teams / 16 and 16
        adds = 32 + rows
        dw_tol = adds * U32 * (np.abs(dy) * h).sum(0) + (np.abs(dy) * h_tol).sum(0)
        db_tol = adds * U32 * np.abs(dy).sum(0)
        DX = Matrix(dev, kind, rows, cols, cols + 1, 7)
        DW, DB = (Raw(dev, np.zeros(cols, ref.STORED[params])) for _ in range(2))
        args = dict(eps=eps, mean=M if given else None, rstd=R if given else None, dtype=kind, param_dtype=params,
                    grad_stride=DY.stride, x_stride=X.stride)
        dev.flayernorm_grad(DY, X, W, DX, DW, DB, rows, cols, dx_stride=DX.stride, **args)
        close(DX.values(), dx, dx_tol * (1 + HALF_STEP[kind]) + stored_tolerance(dx, kind), "dx")
        got_dw, got_db = ref.widen(DW.values(), params), ref.widen(DB.values(), params)
        close(got_dw, dw, dw_tol * 1.01 + stored_tolerance(dw, params), "dweight")
        close(got_db, db, db_tol * 1.01 + stored_tolerance(db, params), "dbias")
        # each output by itself gives the same bits
        first = DX.values()
        D2, W2, B2 = Matrix(dev, kind, rows, cols, cols, 0), Raw(dev, np.zeros(cols, ref.STORED[params])), \
            Raw(dev, np.zeros(cols, ref.STORED[params]))
        dev.flayernorm_grad(DY, X, W, D2, None, None, rows, cols, **args)
        dev.flayernorm_grad(DY, X, W, None, W2, None, rows, cols, **args)
        dev.flayernorm_grad(DY, X, W, None, None, B2, rows, cols, **args)
        assert np.array_equal(D2.values(), first)
        assert np.array_equal(W2.values(), DW.values()) and np.array_equal(B2.values(), DB.values())
        # over dy, and over x
        for over in (Matrix(dev, kind, rows, cols, cols, 0, dy), Matrix(dev, kind, rows, cols, cols, 0, x)):
            is_dy = np.array_equal(over.values(), dy)
            a = dict(args, **({"grad_stride": cols} if is_dy else {"x_stride": cols}))
            dev.flayernorm_grad(over if is_dy else DY, X if is_dy else over, W, over, W2, B2, rows, cols, **a)
            assert np.array_equal(over.values(), first)
            assert np.array_equal(W2.values(), DW.values()) and np.array_equal(B2.values(), DB.values())
            over.free()
        for t in (DX, DW, DB, D2, W2, B2):
            t.free()
    for t in (DY, X, W, M, R):
        t.free()


def test_layernorm_far_from_zero_and_constant_rows(dev):
    """Rows around 1000 with a spread of 1: a mean of squares would lose every digit.  Constant rows: the variance is zero and
    y is the bias."""
    _say("flayernorm offset rows")
    rng = np.random.default_rng(3)
    rows, cols = 6, 1500
    x = ref.rounded(rng.standard_normal((rows, cols)) + 1000, "f32")
    x[2] = 7.5
    x[4] = 0.0
    w, b = ref.rounded(1 + rng.standard_normal(cols), "f32"), ref.rounded(rng.standard_normal(cols), "f32")
    X, Y = Matrix(dev, "f32", rows, cols, values=x), Matrix(dev, "f32", rows, cols)
    W, B = Raw(dev, w.astype(np.float32)), Raw(dev, b.astype(np.float32))
    dev.flayernorm(X, W, B, Y, rows, cols, eps=1e-5)
    y, mean, rstd = ref.layernorm(x, w, b, 1e-5)
    got = Y.values()
    tol = norm_tolerances(x, w, b, y, mean, rstd, "f32")[0]
    close(got, y, tol, "y")
    assert np.array_equal(got[4], b)
    for t in (X, Y, W, B):
        t.free()


def test_layernorm_keeps_nan_and_infinity_in_their_rows(dev):
    _say("flayernorm nan")
    rng = np.random.default_rng(5)
    for cols in (40, 900, 5000, 20000):
        x = ref.rounded(rng.standard_normal((9, cols)), "bf16")
        clean = x.copy()
        x[3, cols // 2] = np.nan
        x[6, 0] = np.inf
        X, Y = Matrix(dev, "bf16", 9, cols, values=x), Matrix(dev, "bf16", 9, cols)
        Z, C = Matrix(dev, "bf16", 9, cols), Matrix(dev, "bf16", 9, cols, values=clean)
        dev.flayernorm(X, None, None, Y, 9, cols, dtype="bf16")
        dev.flayernorm(C, None, None, Z, 9, cols, dtype="bf16")
        got, want = Y.values(), Z.values()
        assert np.isnan(got[3]).all() and np.isnan(got[6]).any()
        others = [0, 1, 2, 4, 5, 7, 8]
        assert np.array_equal(got[others], want[others])
        for t in (X, Y, Z, C):
            t.free()


def test_layernorm_grad_over_no_rows_gives_zeros(dev):
    _say("flayernorm_grad no rows")
    for params in ("f32", "f16", "bf16"):
        kind = "f32" if params == "f32" else params
        DW, DB = (Raw(dev, np.ones(100, ref.STORED[params])) for _ in range(2))
        dev.flayernorm_grad(None, None, None, None, DW, DB, 0, 100, dtype=kind, param_dtype=params)
        assert not DW.values().any() and not DB.values().any()
        DW.free(), DB.free()


# ---- log probabilities ------------------------------------------------------------
# Additions a term passes through: 32 in a tile, up to 16 tiles, six in the wave, four
# waves, up to 24 parts at these sizes; exponent and logarithm add a few more: 128.
# An exponent z is off by 3 u |z| (scale * log2 e, product), which weighs as
# mean_size = sum p |z| in the sums.
TERMS = 128


def logprob_tolerances(r):
    sums = U32 * (TERMS + 4 * r["mean_size"])
    logsum = r["stats"][:, 1]
    with np.errstate(invalid="ignore"):
        logsum_tol = sums + 2 * U32 * np.abs(logsum)
        lp_tol = logsum_tol[:, None] + 3 * U32 * np.abs(r["z"]) + 2 * U32 * np.abs(r["lp"])
        entropy_tol = sums * (2 + r["mean_size"]) + 4 * U32 * np.abs(logsum)
    return logsum_tol, lp_tol, entropy_tol


def check_logprob(dev, x, tokens, kind, scale, top, token_dtype="i64", stride=None, offset=0, parts=True):
    rows, cols = x.shape
    r = ref.logprob(x, tokens, scale, top)
    X = Matrix(dev, kind, rows, cols, stride, offset, x)
    T = Raw(dev, np.asarray(tokens).astype({"i64": np.int64, "i32": np.int32, "f32": np.float32}[token_dtype]))
    LP, H = Raw(dev, np.full(rows, 9, np.float32)), Raw(dev, np.full(rows, 9, np.float32))
    S = Raw(dev, np.full((rows, 2), 9, np.float32))
    TI, TL = Raw(dev, np.full((rows, top), -9, np.int32)), Raw(dev, np.full((rows, top), 9, np.float32))
    dev.flogprob(X, T, LP, rows, cols, scale=scale, stats=S, entropy=H, top=top, top_index=TI, top_logprob=TL, dtype=kind,
                 token_dtype=token_dtype, stride=X.stride)
    logsum_tol, lp_tol, entropy_tol = logprob_tolerances(r)
    with np.errstate(over="ignore"):   # what fp32 does not hold is -infinity
        r.update({k: r[k].astype(np.float32).astype(np.float64) for k in ("logprob", "top_logprob")})
    stats = S.values()
    assert np.array_equal(stats[:, 0], r["stats"][:, 0])
    close(stats[:, 1], r["stats"][:, 1], logsum_tol, "logsum")
    close(H.values(), r["entropy"], entropy_tol, "entropy")
    given_tol = lp_tol[np.arange(rows), np.clip(tokens, 0, cols - 1)]
    close(LP.values(), r["logprob"], given_tol, "logprob")
    if top:
        assert np.array_equal(TI.values(), r["top_index"]), "top_index"
        close(TL.values(), r["top_logprob"], np.take_along_axis(lp_tol, r["top_index"], 1), "top_logprob")
    X.values()
    if parts:  # each output by itself: the same bits
        L2, H2, S2 = Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros((rows, 2), np.float32))
        I2, P2 = Raw(dev, np.zeros((rows, top), np.int32)), Raw(dev, np.zeros((rows, top), np.float32))
        a = dict(scale=scale, dtype=kind, token_dtype=token_dtype, stride=X.stride)
        dev.flogprob(X, T, L2, rows, cols, **a)
        dev.flogprob(X, None, None, rows, cols, entropy=H2, **a)
        dev.flogprob(X, None, None, rows, cols, stats=S2, **a)
        dev.flogprob(X, None, None, rows, cols, top=top, top_index=I2, top_logprob=P2, **a)
        for one, whole in ((L2, LP), (H2, H), (S2, S), (I2, TI), (P2, TL)):
            assert np.array_equal(one.values(), whole.values(), equal_nan=one.array.dtype.kind == "f")
        for t in (L2, H2, S2, I2, P2):
            t.free()
    for t in (X, T, LP, H, S, TI, TL):
        t.free()
    return r


LOGPROB_SHAPES = [(1, 1), (3, 2), (2, 5), (5, 31), (4, 32), (3, 100), (2, 255), (3, 1000), (2, 4096), (3, 4097), (2, 8191),
                  (1, 8193), (4, 10007), (2, 32768), (1, 50021), (3, 65537), (1, 131072), (2, 150000), (1, 300007)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", LOGPROB_SHAPES)
def test_logprob(dev, rows, cols, kind):
    _say("flogprob", rows, cols, kind)
    rng = np.random.default_rng(cols + rows)
    x = ref.rounded(rng.standard_normal((rows, cols)) * 2.5, kind)
    tokens = rng.integers(0, cols, rows)
    for top, scale, stride, offset, token_dtype in ((min(20, cols), 1.0, cols, 0, "i64"), (0, 0.7, cols + 3, 1, "i32"),
                                                    (1, 1.6, cols + 8, 4, "f32"), (min(32, cols), 1.25, cols + 1, 7, "i64")):
        check_logprob(dev, x, tokens, kind, scale, top, token_dtype, stride, offset)
        tokens = rng.integers(0, cols, rows)
        tokens[rng.integers(rows)] = -1


@pytest.mark.parametrize("rows", [300, 1100])
def test_logprob_many_rows(dev, rows):
    _say("flogprob many rows", rows)
    rng = np.random.default_rng(rows)
    for cols, kind, top in ((50, "f32", 7), (3001, "bf16", 32), (9001, "f16", 3)):
        x = ref.rounded(rng.standard_normal((rows, cols)) * 2, kind)
        check_logprob(dev, x, rng.integers(-1, cols, rows), kind, 1.0, top, stride=cols + 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [40, 5000, 70001, 140000])
def test_logprob_ties_masks_and_orders(dev, kind, cols):
    """Alternatives where many logits are equal, sorted, or ruled out: the lowest place first, whatever the order in memory."""
    _say("flogprob orders", kind, cols)
    rng = np.random.default_rng(cols)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": ref.widen(np.array([0xFF7F], np.uint16), "bf16")[0]}[kind]
    rows = [
        np.zeros(cols),                                        # all equal
        np.where(np.arange(cols) % 2, 0.0, -0.0),              # zeros of both signs are equal
        np.linspace(-8, 8, cols), np.linspace(8, -8, cols),    # sorted: the best lie together
        np.floor(rng.standard_normal(cols)),                   # a handful of values
        np.full(cols, -np.inf),                                # nothing is left
        np.where(np.arange(cols) == cols - 1, 1.5, -np.inf),   # one is left, the last
        np.where(rng.random(cols) < 0.001, 2.0, -np.inf),
        np.full(cols, low), np.where(np.arange(cols) == cols // 2, -3.0, low),
        np.where(np.arange(cols) % 8192 < 32, 5.0 + np.arange(cols) / cols, rng.standard_normal(cols)),  # one lane holds the best
        np.where(np.arange(cols) >= cols - 7, 4.0, 3.0),
    ]
    x = ref.rounded(np.stack(rows), kind)
    tokens = np.array([0, cols - 1, 3, 1, 2, 7, cols - 1, 5, 9, cols // 2, 8, cols - 2])
    for top in (1, 5, 32):
        check_logprob(dev, x, tokens, kind, 1.0, top, parts=top == 5)
    check_logprob(dev, x[:8], tokens[:8], kind, 1.5, 20, stride=cols + 1, offset=3, parts=False)


def test_logprob_of_large_logits_loses_nothing(dev):
    """Logits around 10000: their distances count, not their size."""
    _say("flogprob large logits")
    rng = np.random.default_rng(8)
    x = ref.rounded(rng.standard_normal((3, 20011)) * 2 + np.array([[1e4], [-3e4], [9e5]]), "f32")
    check_logprob(dev, x, rng.integers(0, 20011, 3), "f32", 1.0, 9)
    check_logprob(dev, x, rng.integers(0, 20011, 3), "f32", 0.9, 2)


@pytest.mark.parametrize("scale", [2.0 ** -64, 1e-6, 1e6, 2.0 ** 64])
def test_logprob_with_extreme_scales(dev, scale):
    """Almost uniform, and all on the largest: products with the scale may pass what fp32 holds."""
    _say("flogprob scale", scale)
    rng = np.random.default_rng(17)
    x = ref.rounded(rng.standard_normal((4, 9001)) * 3, "f32")
    x[1] = ref.rounded(rng.standard_normal(9001) * 1e30, "f32")
    x[2] = ref.rounded(-np.abs(rng.standard_normal(9001)) * 1e12, "f32")
    check_logprob(dev, x, np.argmax(x, 1), "f32", scale, 4)


@pytest.mark.parametrize("cols", [37, 6000, 140001])
def test_logprob_of_rows_with_nan_infinity_and_wrong_tokens(dev, cols):
    _say("flogprob nan", cols)
    rng = np.random.default_rng(6)
    x = ref.rounded(rng.standard_normal((6, cols)), "f32")
    x[1, cols // 3] = np.nan
    x[3, cols - 1] = np.inf
    x[5] = np.nan
    top = 4
    X, T = Matrix(dev, "f32", 6, cols, values=x), Raw(dev, np.array([cols, 0, cols - 1, 0, 1 << 40, 0], np.int64))
    LP, H, S = Raw(dev, np.zeros(6, np.float32)), Raw(dev, np.zeros(6, np.float32)), Raw(dev, np.zeros((6, 2), np.float32))
    TI, TL = Raw(dev, np.zeros((6, top), np.int32)), Raw(dev, np.zeros((6, top), np.float32))
    dev.flogprob(X, T, LP, 6, cols, stats=S, entropy=H, top=top, top_index=TI, top_logprob=TL)
    lp, h, s, ti, tl = (t.values() for t in (LP, H, S, TI, TL))
    bad = [1, 3, 5]
    assert np.isnan(lp[bad]).all() and np.isnan(h[bad]).all() and np.isnan(s[bad, 1]).all()
    assert (ti[bad] == -1).all() and np.isnan(tl[bad]).all()
    assert np.isnan(lp[[0, 4]]).all()          # no such token
    good = [0, 2, 4]
    r = ref.logprob(x[good], np.array([0, cols - 1, 0]), 1.0, top)
    _, lp_tol, entropy_tol = logprob_tolerances(r)
    assert np.array_equal(ti[good], r["top_index"])
    close(h[good], r["entropy"], entropy_tol, "entropy")
    close(lp[2], r["logprob"][1], lp_tol[1, cols - 1], "logprob")
    D, G = Matrix(dev, "f32", 6, cols), Raw(dev, np.ones(6, np.float32))
    dev.flogprob_grad(X, T, S, G, D, 6, cols)
    d = D.values()
    assert np.isnan(d[[0, 4]]).all() and np.isnan(d[1]).all() and np.isfinite(d[2]).all()
    for t in (X, T, LP, H, S, TI, TL, D, G):
        t.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (4, 37), (5, 1000), (3, 2048), (2, 4095), (4, 10007), (2, 40001), (700, 129)])
def test_logprob_grad(dev, rows, cols, kind):
    _say("flogprob_grad", rows, cols, kind)
    rng = np.random.default_rng(rows + 7 * cols)
    x = ref.rounded(rng.standard_normal((rows, cols)) * 2.5, kind)
    if cols > 30:
        x[rng.random(x.shape) < 0.3] = -np.inf
        x[rows // 2] = -np.inf
    tokens = rng.integers(-1, cols, rows)
    scale = 1.25
    with np.errstate(invalid="ignore"):
        r = ref.logprob(x, tokens, scale)
    # what the pass before left, in fp32
    S = Raw(dev, r["stats"].astype(np.float32))
    H = Raw(dev, r["entropy"].astype(np.float32))
    g, h = ref.rounded(rng.standard_normal(rows), "f32"), ref.rounded(0.1 * rng.standard_normal(rows), "f32")
    G, DH = Raw(dev, g.astype(np.float32)), Raw(dev, h.astype(np.float32))
    for stride, offset, use_g, use_h, token_dtype in ((cols, 0, True, False, "i64"), (cols + 3, 1, True, True, "f32"),
                                                      (cols + 1, 2, False, True, "i32")):
        gg, hh = g * use_g, h * use_h
        d, p = ref.logprob_grad(x, tokens, scale, gg, hh, r)
        # p: its exponent is off by a few u of its terms and by the rounding of logsum
        with np.errstate(invalid="ignore"):
            rel = U32 * (6 * np.abs(np.where(p > 0, r["z"], 0)) + 6 * np.abs(np.where(np.isinf(r["stats"][:, 1:]), 0, r["stats"][:, 1:])) + 8)
            lp = np.where(p > 0, np.abs(r["lp"]), 0) + r["entropy"][:, None]
        tol = scale * (p * rel * (np.abs(gg)[:, None] + lp * np.abs(hh)[:, None]) + p * rel * np.abs(hh)[:, None]
                       + 3 * U32 * (p + 1) * np.abs(gg)[:, None] * (p > 0)) + 4 * U32 * np.abs(d)
        X = Matrix(dev, kind, rows, cols, stride, offset, x)
        T = Raw(dev, tokens.astype({"i64": np.int64, "i32": np.int32, "f32": np.float32}[token_dtype]))
        D = Matrix(dev, kind, rows, cols, stride + 2, offset + 3)
        a = dict(scale=scale, entropy=H if use_h else None, dentropy=DH if use_h else None, dtype=kind, token_dtype=token_dtype,
                 stride=X.stride)
        dev.flogprob_grad(X, T, S, G if use_g else None, D, rows, cols, dlogits_stride=D.stride, **a)
        got = D.values()
        close(got, d, tol * (1 + HALF_STEP[kind]) + stored_tolerance(d, kind), "dlogits")
        X.values()
        dev.flogprob_grad(X, T, S, G if use_g else None, X, rows, cols, dlogits_stride=X.stride, **a)   # in place
        X.whole, was = X.whole.copy(), X.whole
        assert np.array_equal(X.values(), got)
        X.whole = was
        for t in (X, T, D):
            t.free()
    for t in (S, H, G, DH):
        t.free()


@pytest.mark.parametrize("rows,cols,kind", [(1, 5, "f32"), (3, 70001, "bf16"), (700, 129, "f16"), (2, 300007, "f32")])
def test_logprob_grad_computes_missing_stats(dev, rows, cols, kind):
    """Without the forward pass's stats the same bits come out."""
    _say("flogprob_grad without stats", rows, cols, kind)
    rng = np.random.default_rng(cols)
    x = ref.rounded(rng.standard_normal((rows, cols)) * 2, kind)
    X, T = Matrix(dev, kind, rows, cols, cols + 1, 1, x), Raw(dev, rng.integers(-1, cols, rows).astype(np.int64))
    S, H, G = Raw(dev, np.zeros((rows, 2), np.float32)), Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.full(rows, -0.5, np.float32))
    one, other = Matrix(dev, kind, rows, cols), Matrix(dev, kind, rows, cols)
    a = dict(dtype=kind, stride=X.stride, scale=1.5)
    dev.flogprob(X, None, None, rows, cols, stats=S, entropy=H, **a)
    for entropy in (None, H):
        dev.flogprob_grad(X, T, S, G, one, rows, cols, entropy=entropy, dentropy=entropy and G, **a)
        dev.flogprob_grad(X, T, None, G, other, rows, cols, entropy=entropy, dentropy=entropy and G, **a)
        assert np.array_equal(one.values(), other.values())
    for t in (X, T, S, H, G, one, other):
        t.free()


def test_logprob_of_more_rows_than_a_launch_takes(dev):
    """One logit per row: log probability and gradient are 0; more work-groups than one launch has."""
    _say("flogprob 8.5 million rows")
    rows = (1 << 23) + 12345
    x = np.random.default_rng(1).standard_normal(rows).astype(np.float32)
    X, T = Raw(dev, x), Raw(dev, np.zeros(rows, np.int32))
    LP, S, G = Raw(dev, np.ones(rows, np.float32)), Raw(dev, np.ones((rows, 2), np.float32)), Raw(dev, np.ones(rows, np.float32))
    TI, TL = Raw(dev, np.full(rows, 9, np.int32)), Raw(dev, np.ones(rows, np.float32))
    dev.flogprob(X, T, LP, rows, 1, stats=S, top=1, top_index=TI, top_logprob=TL, token_dtype="i32")
    # the sum is one exponential of (almost) 0 times another: each within a unit in the last place (2 u) of 1, the
    # product rounds once more, and the logarithm of 1 + 5 u within its own last place: 8 u of 0
    s = S.values()
    assert not TI.values().any() and np.array_equal(s[:, 0], x)
    for v in (LP.values(), TL.values(), s[:, 1]):
        assert np.abs(v).max() <= 8 * U32
    dev.flogprob_grad(X, T, S, G, X, rows, 1, token_dtype="i32")
    # p is e to the power of that, with one more exponential's 2 u: 1 - p is off by 8 u + 2 u and two roundings
    assert np.abs(X.values()).max() <= 12 * U32
    for t in (X, T, LP, S, G, TI, TL):
        t.free()


def test_logprob_grad_against_differences_of_the_forward_pass(dev):
    """dlogits of the device against central differences of the 64-bit forward pass."""
    _say("flogprob_grad differences")
    rng = np.random.default_rng(12)
    x = ref.rounded(rng.standard_normal((3, 11)), "f32")
    tokens, g, h = np.array([4, 0, 10]), np.array([1.0, -0.5, 2.0]), np.array([0.25, 1.0, -0.5])
    X, T = Matrix(dev, "f32", 3, 11, values=x), Raw(dev, tokens.astype(np.int64))
    LP, H, S = Raw(dev, np.zeros(3, np.float32)), Raw(dev, np.zeros(3, np.float32)), Raw(dev, np.zeros((3, 2), np.float32))
    G, DH, D = Raw(dev, g.astype(np.float32)), Raw(dev, h.astype(np.float32)), Matrix(dev, "f32", 3, 11)
    dev.flogprob(X, T, LP, 3, 11, stats=S, entropy=H)
    dev.flogprob_grad(X, T, S, G, D, 3, 11, entropy=H, dentropy=DH)
    got = D.values()
    for i in np.ndindex(x.shape):
        sides = []
        for step in (1e-5, -1e-5):
            y = x.copy()
            y[i] += step
            r = ref.logprob(y, tokens, 1.0)
            sides.append((r["logprob"] * g + r["entropy"] * h).sum())
        want = (sides[0] - sides[1]) / 2e-5
        # fp32 results of about ten roundings on values up to 5; the differences are good to 1e-9
        assert abs(got[i] - want) <= 20 * U32 * 5, (i, got[i], want)
    for t in (X, T, LP, H, S, G, DH, D):
        t.free()


@pytest.mark.parametrize("rows", [1, 8, 40])
def test_logprob_calls_in_a_row_take_nothing_from_each_other(dev, rows):
    """Rows in parts meet in a workspace that every call uses again: 200 calls on two inputs in turn, some with a product that
    splits its contraction (the same workspace and counters) between them, each compared with the first of its kind."""
    _say("flogprob repeated", rows)
    rng = np.random.default_rng(rows)
    cols, top = 60011, 11
    X = [Matrix(dev, "bf16", rows, cols, values=rng.standard_normal((rows, cols))) for _ in range(2)]
    T = Raw(dev, rng.integers(0, cols, rows).astype(np.int64))
    outs = [[Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros(rows, np.float32)), Raw(dev, np.zeros((rows, 2), np.float32)),
             Raw(dev, np.zeros((rows, top), np.int32)), Raw(dev, np.zeros((rows, top), np.float32))] for _ in range(4)]
    a, b = dev.array(np.ones(96 * 8192)), dev.array(np.ones(96 * 8192))
    c = dev.empty(96 * 96)

    def call(i, o):
        dev.flogprob(X[i], T, o[0], rows, cols, entropy=o[1], stats=o[2], top=top, top_index=o[3], top_logprob=o[4], dtype="bf16")
    for i in range(2):
        call(i, outs[i])
    want = [[t.values() for t in o] for o in outs[:2]]
    for n in range(100):
        for i in range(2):
            call(i, outs[2 + i])
        if n % 7 == 0:
            dev.fmatmul(False, True, a, b, c, 96, 96, 8192)
        if n % 10 == 0:
            for i in range(2):
                for t, w in zip(outs[2 + i], want[i]):
                    assert np.array_equal(t.values(), w)
    assert np.all(c.download() == 8192)
    for t in [*X, T, a, b, c, *(t for o in outs for t in o)]:
        t.free()


def test_two_threads_call_one_device(dev):
    """Calls of two threads on one handle that use its workspace: each thread's results are its own."""
    _say("two threads")
    import threading
    rng = np.random.default_rng(3)
    rows, cols = 5, 40000
    jobs = []
    for i in range(2):
        x = ref.rounded(rng.standard_normal((rows, cols)), "f32")
        dy = ref.rounded(rng.standard_normal((64, 300)), "f32")
        jobs.append(dict(X=Matrix(dev, "f32", rows, cols, values=x), TI=Raw(dev, np.zeros((rows, 6), np.int32)),
                         TL=Raw(dev, np.zeros((rows, 6), np.float32)), want=ref.logprob(x, np.zeros(rows, int), 1.0, 6)["top_index"],
                         DY=Matrix(dev, "f32", 64, 300, values=dy), DB=Raw(dev, np.zeros(300, np.float32)), db=dy.sum(0), bad=[]))

    def work(j):
        for _ in range(60):
            dev.flogprob(j["X"], None, None, rows, cols, top=6, top_index=j["TI"], top_logprob=j["TL"])
            dev.flayernorm_grad(j["DY"], j["DY"], None, None, None, j["DB"], 64, 300)
            if not np.array_equal(j["TI"].values(), j["want"]) or np.abs(j["DB"].values() - j["db"]).max() > 1e-4:
                j["bad"].append(1)
    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not jobs[0]["bad"] and not jobs[1]["bad"]
    for j in jobs:
        for k in ("X", "TI", "TL", "DY", "DB"):
            j[k].free()


def test_rows_whose_offsets_pass_32_bits(dev):
    """Three rows 2^31 + 5 elements apart (8.6 GB): every row is read and written where it lies."""
    _say("far rows")
    rng = np.random.default_rng(9)
    cols, stride = 5003, (1 << 31) + 5
    base = dev.alloc_bytes(2 * (2 * stride + cols + 8))
    x = ref.rounded(rng.standard_normal((3, cols)), "bf16")

    def put(values):
        for i in range(3):
            row = ref.store(values[i], "bf16")
            dev.copy_to_device(base + 2 * i * stride, row.ctypes.data, row.nbytes)

    def get():
        out = np.empty((3, cols), np.uint16)
        for i in range(3):
            dev.copy_to_host(out[i].ctypes.data, base + 2 * i * stride, out[i].nbytes)
        return ref.widen(out, "bf16")
    N, T = Matrix(dev, "bf16", 3, cols, values=x), Raw(dev, np.array([1, 2, cols - 1], np.int64))
    S, G = [Raw(dev, np.zeros((3, 2), np.float32)) for _ in range(2)], Raw(dev, np.ones(3, np.float32))
    I, P = [Raw(dev, np.zeros((3, 4), np.int32)) for _ in range(2)], Raw(dev, np.zeros((3, 4), np.float32))
    for at, st, s, i in ((base, stride, S[0], I[0]), (N, cols, S[1], I[1])):
        put(x)
        dev.flogprob(at, T, None, 3, cols, stats=s, top=4, top_index=i, top_logprob=P, dtype="bf16", stride=st)
        dev.flogprob_grad(at, T, s, G, at, 3, cols, dtype="bf16", stride=st, dlogits_stride=st)
        dev.flayernorm(at, None, None, at, 3, cols, dtype="bf16", x_stride=st, out_stride=st)
        dev.flayernorm_grad(at, at, None, at, None, None, 3, cols, dtype="bf16", x_stride=st, grad_stride=st, dx_stride=st)
        if at == base:
            far = get()
    N.whole = N._download()   # what was written in place is checked against the far rows, not against the start
    near = N.values()
    assert np.array_equal(far, near) and np.isfinite(far).all() and far.any()
    assert np.array_equal(S[0].values(), S[1].values()) and np.array_equal(I[0].values(), I[1].values())
    dev._free(base)
    dev.pool_trim()
    for t in (N, T, G, P, *S, *I):
        t.free()


# ---- AdamW ------------------------------------------------------------------------

ADAMW = dict(lr=2e-3, beta1=0.9, beta2=0.999, eps=1e-8)
ADAMW_SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 1023, 4096, 4097, 10000, 0, 65536 + 13, 7]


def adamw_tolerances(p, g, m0, v0, new_p, new_m, new_v, wd):
    m_tol = 4 * U32 * (np.abs(m0) + np.abs(g)) + 2.0 ** -140
    v_tol = 6 * U32 * np.abs(new_v) + 2.0 ** -140
    update = np.abs(p - ADAMW["lr"] * wd * p - new_p)
    # m_tol over the same divisor, and eight roundings of the quotient's own
    m_part = np.where(np.abs(new_m) > 0, m_tol / np.maximum(np.abs(new_m), 1e-300), 0)
    p_tol = 4 * U32 * np.abs(p) + update * (12 * U32 + np.minimum(m_part, 1e6)) + 2.0 ** -140
    return p_tol, m_tol, v_tol


@pytest.mark.parametrize("kind,grad", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f16", "f16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("state", ["f32", "8bit"])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw(dev, kind, grad, state, offset):
    """A list of tensors of all sizes, longer than one launch takes; nothing behind a tensor is written."""
    _say("fadamw", kind, grad, state, offset)
    rng = np.random.default_rng(77 + offset)
    sizes = ADAMW_SIZES * 4 if state == "f32" else ADAMW_SIZES * 3
    seed, step, scale = 12345, 7, 0.5
    made, fields, first = [], [], 0
    for i, n in enumerate(sizes):
        p = ref.rounded(rng.standard_normal(n) * 0.1, "f32")
        g = ref.rounded(rng.standard_normal(n) * 10.0 ** rng.integers(-4, 1), grad)
        if n > 600:
            g[300:560] = 0.0
        wd = 0.1 * (i % 2)
        t = dict(n=n, p=p, g=g, wd=wd, first=first)
        t["G"] = Matrix(dev, grad, 1, n, n + 1, offset, g)
        t["P"] = Matrix(dev, kind, 1, n, n + 1, offset, p if kind == "f32" else np.zeros(n))
        t["MASTER"] = Matrix(dev, "f32", 1, n, n + 1, offset, p) if kind != "f32" else None
        if state == "f32":
            t["m"], t["v"] = ref.rounded(rng.standard_normal(n) * 0.05, "f32"), ref.rounded(rng.random(n) * 0.01, "f32")
            t["M"], t["V"] = Matrix(dev, "f32", 1, n, n + 1, offset, t["m"]), Matrix(dev, "f32", 1, n, n + 1, offset, t["v"])
            t["MS"] = t["VS"] = None
        else:
            blocks = max(1, -(-n // 256))
            codes_m, codes_v = rng.integers(0, 256, n).astype(np.uint8), rng.integers(0, 127, n).astype(np.uint8)
            codes_m[(codes_m & 0x7F) == 0x7F] = 3
            ms = (rng.random(blocks) * 1e-3).astype(np.float32)
            vs = (rng.random(blocks) * 1e-3).astype(np.float32)
            ms[0] *= i % 3 != 0  # a block that is zero
            by = np.arange(n) // 256
            t["m"] = ref.E4M3[codes_m] * ms[by].astype(np.float64)
            t["v"] = (ref.E4M3[codes_v] * vs[by].astype(np.float64)) ** 2
            pad = np.zeros(offset, np.uint8)
            t["M"], t["V"] = Raw(dev, np.concatenate([pad, codes_m])), Raw(dev, np.concatenate([pad, codes_v]))
            t["MS"], t["VS"] = Raw(dev, ms), Raw(dev, vs)
        fields.append(dict(count=n, first=first, weight_decay=wd, param=t["P"], grad=t["G"], master=t["MASTER"],
                           m=t["M"] if state == "f32" else t["M"].ptr + offset, v=t["V"] if state == "f32" else t["V"].ptr + offset,
                           m_scale=t["MS"], v_scale=t["VS"]))
        made.append(t)
        first += n
    dev.fadamw(capi.adamw_tensors(fields), step=step, seed=seed, dtype=kind, grad_dtype=grad, state_dtype=state, grad_scale=scale,
               **ADAMW)
    for t in made:
        n, p, g, wd = t["n"], t["p"], t["g"], t["wd"]
        new_p, new_m, new_v = ref.adamw(p, g, t["m"], t["v"], wd, step, grad_scale=scale, **ADAMW)
        p_tol, m_tol, v_tol = adamw_tolerances(p, g * scale, t["m"], t["v"], new_p, new_m, new_v, wd)
        if kind == "f32":
            close(t["P"].values()[0], new_p, p_tol, "param")
        else:
            master = t["MASTER"].values()[0]
            close(master, new_p, p_tol, "master")
            assert np.array_equal(t["P"].values()[0], ref.rounded(master, kind))
        assert np.array_equal(t["G"].values()[0], g)
        if state == "f32":
            close(t["M"].values()[0], new_m, m_tol, "m")
            close(t["V"].values()[0], new_v, v_tol, "v")
        elif n:
            bits = ref.random_bits(seed, t["first"] + np.arange(n))
            for codes, scales, new, random, rel in ((t["M"], t["MS"], new_m, bits & np.uint64(0xFFFF), m_tol),
                                                    (t["V"], t["VS"], np.sqrt(new_v), bits >> np.uint64(16), 4 * U32 * np.sqrt(new_v))):
                largest = ref.block_largest(new)
                got_scale = scales.values().astype(np.float64)
                top_tol = np.array([rel[b * 256:(b + 1) * 256].max() for b in range(largest.size)])
                close(got_scale, largest / 448, (top_tol + 3 * U32 * largest) / 448, "scale")
                by = np.arange(n) // 256
                live = largest[by] > 0
                got = ref.E4M3[codes.values()[offset:]]
                scale_of = np.where(live, got_scale[by], 1.0)
                at, unit = ref.held_in_8_bits(new, scale_of, random.astype(np.float64))
                # where the value lies so near a border that fp32 may fall on either side, either neighbour is right
                near = (rel / scale_of + 6 * U32 * np.abs(new) / scale_of) / unit + 2.0 ** -20
                low, high = np.floor(at - near) * unit, np.floor(at + near) * unit
                size = np.where(live, np.abs(got), 0)
                assert ((size >= np.minimum(low, 448)) & (size <= np.minimum(high, 448)))[live].all()
                assert (got[~live] == 0).all()
                signed = live & (size > 0)
                assert (np.sign(got[signed]) == np.sign(new[signed])).all()
    for t in made:
        for k in ("G", "P", "MASTER", "M", "V", "MS", "VS"):
            if t[k] is not None:
                t[k].free()


def test_adamw_8_bit_states_follow_on_average(dev):
    """v moves by a thousandth of its distance per step, far less than half a step of an 8-bit float: only because the
    rounding is stochastic does it move at all.  After 1000 steps with a constant gradient sqrt(v) of 64-bit arithmetic is
    sqrt(1 - 0.999^1000) |g| = 0.795 |g|."""
    _say("fadamw 8 bit long run")
    n = 4096
    rng = np.random.default_rng(2)
    g = ref.rounded(np.where(rng.random(n) < 0.5, 0.5, 1.0) * np.sign(rng.standard_normal(n)), "f32")
    P, G = Raw(dev, np.zeros(n, np.float32)), Raw(dev, g.astype(np.float32))
    M, V = Raw(dev, np.zeros(n, np.uint8)), Raw(dev, np.zeros(n, np.uint8))
    MS, VS = Raw(dev, np.zeros(n // 256, np.float32)), Raw(dev, np.zeros(n // 256, np.float32))
    plan = capi.adamw_tensors([dict(count=n, param=P, grad=G, m=M, v=V, m_scale=MS, v_scale=VS)])
    for step in range(1, 1001):
        dev.fadamw(plan, step=step, lr=1e-3, seed=step, state_dtype="8bit")
    root = ref.E4M3[V.values()] * np.repeat(VS.values().astype(np.float64), 256)
    want = math.sqrt(1 - 0.999 ** 1000)
    # one value scatters by some steps of 6 to 12 %; the mean over 2000 of them by a fraction of a percent.  Squares average
    # higher than the square of the average: v = E[sqrt(v)]^2 + variance, at most (0.12)^2 of it
    for size in (0.5, 1.0):
        mean = (root[np.abs(g) == size] ** 2).mean()
        assert abs(mean / (want * size) ** 2 - 1) < 0.05, (size, mean, (want * size) ** 2)
    for t in (P, G, M, V, MS, VS):
        t.free()


@pytest.mark.parametrize("state", ["f32", "8bit"])
def test_adamw_keeps_nan_and_infinity_in_their_elements(dev, state):
    """A gradient that is not finite spoils its own element, now and in the next step, and no other of its block."""
    _say("fadamw nan", state)
    rng = np.random.default_rng(14)
    n = 1000
    g = rng.standard_normal(n).astype(np.float32) * 0.1
    bad = np.zeros(n, bool)
    bad[[7, 300, 999]] = True
    spoilt = g.copy()
    spoilt[7], spoilt[300], spoilt[999] = np.nan, np.inf, -np.inf
    results = []
    for first in (g, spoilt):
        P = Raw(dev, np.full(n, 0.5, np.float32))
        grads = [Raw(dev, first), Raw(dev, g)]
        code = np.uint8 if state == "8bit" else np.float32
        M, V = Raw(dev, np.zeros(n, code)), Raw(dev, np.zeros(n, code))
        MS, VS = Raw(dev, np.zeros(4, np.float32)), Raw(dev, np.zeros(4, np.float32))
        for step, G in enumerate(grads, 1):
            dev.fadamw(capi.adamw_tensors([dict(count=n, param=P, grad=G, m=M, v=V, m_scale=MS, v_scale=VS)]), step=step, lr=1e-3,
                       seed=step, state_dtype=state)
        results.append((P.values(), MS.values(), VS.values()))
        for t in (P, M, V, MS, VS, *grads):
            t.free()
    (clean, ms, vs), (got, got_ms, got_vs) = results
    assert not np.isfinite(got[bad]).any() and np.isfinite(got[~bad]).all()
    if state == "f32":
        assert np.array_equal(got[~bad], clean[~bad])
    else:
        # the scales lack the spoilt elements, no more; a block without one is as it was
        assert np.isfinite(got_ms).all() and np.isfinite(got_vs).all()
        assert (got_ms <= ms).all() and np.array_equal(got[512:768], clean[512:768])
        # an update is lr in size at most about the first steps: sqrt(v) and m of one gradient; the states' rounding
        # moves it by 1/8 of lr per state
        assert np.abs(got - clean)[~bad].max() <= 0.25e-3


def test_adamw_beyond_32_bit_offsets(dev):
    """A tensor of 2^30 + 1027 fp32 elements (4 GiB a buffer): its last elements are updated like its first."""
    _say("fadamw 2^30 elements")
    n = (1 << 30) + 1027
    bufs = [dev.empty(n) for _ in range(4)]
    for b, v in zip(bufs, (0.5, 0.25, 0.125, 0.0625)):
        dev.ffill(v, b)
    p, g, m, v = bufs
    dev.fadamw(capi.adamw_tensors([dict(count=n - 1, param=p, grad=g, m=m, v=v, weight_decay=0.5)]), step=3, **ADAMW)
    new = ref.adamw(0.5, 0.25, 0.125, 0.0625, 0.5, 3, grad_scale=1.0, **ADAMW)
    for buf, want, old in ((p, new[0], 0.5), (m, new[1], 0.125), (v, new[2], 0.0625)):
        for at in (0, 1 << 29, n - 1000):
            part = np.empty(1000, np.float32)
            dev.copy_to_host(part.ctypes.data, buf.ptr + 4 * at, part.nbytes)
            if at == n - 1000:
                assert part[-1] == np.float32(old)     # behind the tensor's end
                part = part[:-1]
            assert np.abs(part - want).max() <= 16 * U32 * abs(want)
    for b in bufs:
        b.free()
    dev.pool_trim()


# ---- together ---------------------------------------------------------------------

def test_a_training_step_of_a_normed_classifier(dev):
    """x -> layer norm -> product with W -> log probabilities, the gradients of the mean loss with regard to everything, and an
    AdamW step on norm and W: each gradient against 64 bits, the weights against the step on the device's own gradients."""
    _say("training step")
    rng = np.random.default_rng(21)
    rows, cols, classes = 96, 200, 1003
    x = ref.rounded(rng.standard_normal((rows, cols)), "f32")
    w, b = ref.rounded(1 + 0.1 * rng.standard_normal(cols), "f32"), ref.rounded(0.1 * rng.standard_normal(cols), "f32")
    W = ref.rounded(rng.standard_normal((cols, classes)) / math.sqrt(cols), "f32")
    tokens = rng.integers(0, classes, rows)
    tokens[5] = -1
    counted = rows - 1
    f32 = lambda a: Raw(dev, np.asarray(a, dtype=np.float32))  # noqa: E731
    X, NW, NB, WW, T = f32(x), f32(w), f32(b), f32(W), Raw(dev, tokens.astype(np.int32))
    Y, MEAN, RSTD = f32(np.zeros((rows, cols))), f32(np.zeros(rows)), f32(np.zeros(rows))
    Z, LP, S = f32(np.zeros((rows, classes))), f32(np.zeros(rows)), f32(np.zeros((rows, 2)))
    G = f32(np.full(rows, -1.0 / counted))
    DZ, DW, DY = f32(np.zeros((rows, classes))), f32(np.zeros((cols, classes))), f32(np.zeros((rows, cols)))
    DX, DNW, DNB = f32(np.zeros((rows, cols))), f32(np.zeros(cols)), f32(np.zeros(cols))
    dev.flayernorm(X, NW, NB, Y, rows, cols, mean=MEAN, rstd=RSTD)
    dev.fmatmul(False, False, Y, WW, Z, rows, classes, cols)
    dev.flogprob(Z, T, LP, rows, classes, stats=S, token_dtype="i32")
    dev.flogprob_grad(Z, T, S, G, DZ, rows, classes, token_dtype="i32")
    dev.fmatmul(True, False, Y, DZ, DW, cols, classes, rows)
    dev.fmatmul(False, True, DZ, WW, DY, rows, cols, classes)
    dev.flayernorm_grad(DY, X, NW, DX, DNW, DNB, rows, cols, mean=MEAN, rstd=RSTD)

    y, mean, rstd = ref.layernorm(x, w, b, 1e-5)
    r = ref.logprob(y @ W, tokens, 1.0)
    dz, _ = ref.logprob_grad(y @ W, tokens, 1.0, np.full(rows, -1.0 / counted), np.zeros(rows), r)
    dx, dw, db = ref.layernorm_grad(dz @ W.T, x, w, mean, rstd)
    # the products set the error: 1e-4 of the norm is the framework's bound for them, and each step keeps the relative error
    for got, want, name in ((LP, r["logprob"], "logprob"), (DZ, dz, "dz"), (DW, y.T @ dz, "dW"), (DX, dx, "dx"), (DNW, dw, "dweight"),
                            (DNB, db, "dbias")):
        v = got.values().astype(np.float64)
        assert np.linalg.norm(v - want) <= 1e-4 * np.linalg.norm(want), name
    assert not DZ.values()[5].any() and not DX.values()[5].any()

    grads = [t.values().astype(np.float64).ravel() for t in (DW, DNW, DNB)]
    zeros = [f32(np.zeros(g.size)) for g in grads for _ in range(2)]
    plan = capi.adamw_tensors([dict(count=g.size, weight_decay=wd, param=p, grad=t, m=zeros[2 * i], v=zeros[2 * i + 1])
                               for i, (g, p, t, wd) in enumerate(zip(grads, (WW, NW, NB), (DW, DNW, DNB), (0.1, 0.0, 0.0)))])
    dev.fadamw(plan, step=1, **ADAMW)
    for p, g, was, wd in ((WW, grads[0], W.ravel(), 0.1), (NW, grads[1], w, 0.0), (NB, grads[2], b, 0.0)):
        new_p, new_m, new_v = ref.adamw(was, g, 0.0 * g, 0.0 * g, wd, 1, grad_scale=1.0, **ADAMW)
        tol, _, _ = adamw_tolerances(was, g, 0.0 * g, 0.0 * g, new_p, new_m, new_v, wd)
        close(p.values().ravel(), new_p, tol, "param after a step")
    for t in (X, NW, NB, WW, T, Y, MEAN, RSTD, Z, LP, S, G, DZ, DW, DY, DX, DNW, DNB, *zeros):
        t.free()


def test_calls_on_two_devices_handles_and_shared_workspace(dev):
    """Two handles on one GPU have streams and workspaces of their own; calls of one handle that share its workspace follow
    each other."""
    _say("two handles")
    rng = np.random.default_rng(31)
    rows, cols = 3, 60000
    x = [ref.rounded(rng.standard_normal((rows, cols)), "f32") for _ in range(2)]
    want = [ref.logprob(a, [0, 1, 2], 1.0, 8) for a in x]
    with capi.Device(0) as other:
        sets = []
        for d in (dev, other):
            sets.append([dict(X=Matrix(d, "f32", rows, cols, values=a), TI=Raw(d, np.zeros((rows, 8), np.int32)),
                              TL=Raw(d, np.zeros((rows, 8), np.float32))) for a in x])
            d.synchronize()
        for _ in range(10):
            for i in range(2):
                for d, s in zip((dev, other), sets):
                    d.flogprob(s[i]["X"], None, None, rows, cols, top=8, top_index=s[i]["TI"], top_logprob=s[i]["TL"])
        for s in sets:
            for i in range(2):
                assert np.array_equal(s[i]["TI"].values(), want[i]["top_index"])
        for s in sets:
            for i in range(2):
                for t in s[i].values():
                    t.free()
