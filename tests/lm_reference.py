"""Plain implementations in 64 bits of the language-model operators, element
types as numpy sees them, and matrices in device memory whose rows lie apart.
Used by the tests only."""
import numpy as np

U32 = 2.0 ** -24  # half a step of fp32, relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}  # steps near zero are no smaller than this
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
STORED = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def to_bf16(x):
    """fp32 -> bf16 bits, to nearest, ties to even."""
    bits = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    rounded = ((bits.astype(np.uint64) + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded).astype(np.uint16)


def store(x, kind):
    with np.errstate(over="ignore"):
        return to_bf16(x) if kind == "bf16" else np.asarray(x).astype(STORED[kind])


def widen(stored, kind):
    """The values that stored elements stand for, in 64 bits."""
    if kind == "bf16":
        return (stored.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return stored.astype(np.float64)


def rounded(x, kind):
    return widen(store(x, kind), kind)


class Matrix:
    """rows x cols in device memory, rows `stride` elements apart, the first one `offset` elements behind a 256-byte
    boundary; what lies between and around the rows is filled with a pattern that untouched() looks for."""

    GUARD = 40

    def __init__(self, dev, kind, rows, cols, stride=None, offset=0, values=None):
        self.dev, self.kind, self.rows, self.cols = dev, kind, rows, cols
        self.stride = cols if stride is None else stride
        self.offset = offset
        n = offset + max(rows, 1) * self.stride + self.GUARD
        self.whole = np.frombuffer(np.random.default_rng(9).bytes(n * SIZE[kind]), dtype=STORED[kind]).copy()
        self.base = dev.alloc_bytes(n * SIZE[kind])
        self.ptr = self.base + offset * SIZE[kind]
        if values is not None:
            self._rows(self.whole)[...] = store(values, kind).reshape(rows, cols)
        dev.copy_to_device(self.base, self.whole.ctypes.data, self.whole.nbytes)

    def _rows(self, whole):
        body = whole[self.offset:self.offset + self.rows * self.stride]
        return body.reshape(self.rows, self.stride)[:, :self.cols]

    def _download(self):
        out = np.empty_like(self.whole)
        self.dev.copy_to_host(out.ctypes.data, self.base, out.nbytes)
        return out

    def values(self):
        """What the rows hold now, in 64 bits; nothing outside them may have changed."""
        now = self._download()
        got = widen(self._rows(now).copy(), self.kind)
        self._rows(now)[...] = self._rows(self.whole)
        assert np.array_equal(now.view(np.uint8), self.whole.view(np.uint8)), "memory outside the rows was written"
        return got

    def free(self):
        self.dev._free(self.base)


class Raw:
    """A flat array of any numpy type in device memory, with a guard behind it."""

    def __init__(self, dev, array):
        self.dev = dev
        self.array = np.ascontiguousarray(array)
        self.guard = np.frombuffer(np.random.default_rng(4).bytes(64), dtype=np.uint8)
        whole = np.concatenate([self.array.reshape(-1).view(np.uint8), self.guard])
        self.ptr = dev.alloc_bytes(whole.nbytes)
        dev.copy_to_device(self.ptr, whole.ctypes.data, whole.nbytes)

    def values(self):
        out = np.empty(self.array.nbytes + 64, dtype=np.uint8)
        self.dev.copy_to_host(out.ctypes.data, self.ptr, out.nbytes)
        assert np.array_equal(out[self.array.nbytes:], self.guard), "memory behind the array was written"
        return out[:self.array.nbytes].view(self.array.dtype).reshape(self.array.shape).copy()

    def free(self):
        self.dev._free(self.ptr)


# ---- layer norm -----------------------------------------------------------------

def layernorm(x, w, b, eps):
    mean = x.mean(1)
    var = ((x - mean[:, None]) ** 2).mean(1)
    rstd = 1 / np.sqrt(var + eps)
    return (x - mean[:, None]) * rstd[:, None] * w + b, mean, rstd


def layernorm_grad(dy, x, w, mean, rstd):
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


# ---- log probabilities ------------------------------------------------------------

def logprob(x, tokens, scale, top=0):
    """dict of logprob, stats, entropy, top_index, top_logprob, and mean_size = sum p |z|, for rows without NaN or +inf."""
    rows = x.shape[0]
    m = x.max(1)
    z = (x - np.where(np.isinf(m), 0.0, m)[:, None]) * scale
    e = np.exp(z)
    s0 = e.sum(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        logsum = np.log(s0)
        size = np.where(e > 0, -z * e, 0.0).sum(1) / np.where(s0 > 0, s0, 1.0)
        entropy = np.where(s0 > 0, logsum + size, 0.0)
        lp = np.where(s0[:, None] > 0, z - logsum[:, None], -np.inf)
    tokens = np.asarray(tokens)
    given = lp[np.arange(rows), np.clip(tokens, 0, x.shape[1] - 1)]
    given = np.where(tokens < 0, 0.0, np.where(tokens >= x.shape[1], np.nan, given))
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return dict(logprob=given, stats=np.stack([m, logsum], 1), entropy=entropy, mean_size=size, z=z, lp=lp,
                top_index=order, top_logprob=np.take_along_axis(lp, order, 1))


def logprob_grad(x, tokens, scale, g, h, r):
    """r: what logprob() gave."""
    rows, cols = x.shape
    tokens = np.asarray(tokens)
    alive = r["stats"][:, 0] > -np.inf
    p = np.where(alive[:, None], np.exp(r["lp"]), 0.0)
    counted = alive & (tokens >= 0)
    d = -p * np.where(counted, g, 0.0)[:, None]
    d[np.arange(rows), np.clip(tokens, 0, cols - 1)] += np.where(counted, g, 0.0)
    with np.errstate(invalid="ignore"):
        d -= np.where(p > 0, p * (r["lp"] + r["entropy"][:, None]), 0.0) * h[:, None]
    return d * scale, p


# ---- AdamW --------------------------------------------------------------------------

E4M3 = np.array([(-1.0 if c & 0x80 else 1.0) * ((c & 7) * 2.0 ** -9 if c & 0x78 == 0 else
                                                (8 + (c & 7)) * 2.0 ** (((c >> 3) & 15) - 10)) for c in range(256)])
E4M3[[0x7F, 0xFF]] = np.nan


def random_bits(seed, elements):
    e = np.asarray(elements, dtype=np.uint64)
    m = np.uint64(0xFFFFFFFF)
    h = ((e & m) * np.uint64(0x9E3779B1) + (e >> np.uint64(32)) * np.uint64(0x6A09E667) + np.uint64(seed)) & m
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & m
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & m
    return h ^ (h >> np.uint64(16))


def adamw(p, g, m, v, wd, step, lr, beta1, beta2, eps, grad_scale):
    g = g * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    update = lr / (1 - beta1 ** step) * m / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return p - lr * wd * p - update, m, v


def block_largest(x, block=256):
    n = -(-x.size // block)
    padded = np.zeros(n * block)
    padded[:x.size] = np.abs(x)
    return padded.reshape(n, block).max(1)


def held_in_8_bits(x, scale, random):
    """(lower code's size in steps of the float's last place plus random / 65536, step): the rounded size is
    floor(first) * step."""
    t = np.abs(x) / scale
    step = 2.0 ** np.maximum(np.floor(np.log2(np.maximum(t, 2.0 ** -20))) - 3, -9)
    return t / step + random / 65536.0, step
