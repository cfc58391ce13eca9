"""What is measured of the operators of a language model's training step and sampling loop: layer norm, log
probabilities of given tokens, and AdamW, each in its plain form (elementary torch operations) and, where `own` is
true, through the framework's entry points.

The framework's device has a stream of its own: inputs are complete before a call (the caller synchronises once after
making them), and outputs go to buffers that the caller holds, as with every builtin of the framework.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 256  # elements that share a scale where AdamW's states are held in 8 bits
MASK32 = 0xFFFFFFFF


# ---- the cases --------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token in each of four sequences: latency
        dict(name="norm 4x4096 bf16", op="layernorm", rows=4, cols=4096, pad=0, type="bf16", params="bf16"),
        # rows of an odd length inside a wider buffer
        dict(name="norm 2049x1021 f16", op="layernorm", rows=2049, cols=1021, pad=6, type="f16", params="f32"),
        # a long batch of a wide model
        dict(name="norm 16384x8192 bf16", op="layernorm", rows=16384, cols=8192, pad=0, type="bf16", params="f32"),
        # a batch of 256 rows of 784 features, as the logistic regression has them
        dict(name="norm grad 256x784 f32", op="layernorm_grad", rows=256, cols=784, pad=0, type="f32", params="f32"),
        # training on a long batch
        dict(name="norm grad 16384x4096 bf16", op="layernorm_grad", rows=16384, cols=4096, pad=0, type="bf16", params="f32"),
        # sampling: eight sequences' next tokens, twenty alternatives each, a temperature of 0.8
        dict(name="logprob 8x131072 bf16 top 20", op="logprob", rows=8, cols=131072, pad=0, type="bf16", top=20, scale=1.25, masked=0.0),
        # scores of a prompt under a grammar that rules most tokens out; odd vocabulary, padded rows
        dict(name="logprob 1024x50021 f32 top 5", op="logprob", rows=1024, cols=50021, pad=3, type="f32", top=5, scale=1.0, masked=0.9),
        # scores of a long batch
        dict(name="logprob 4096x131072 bf16 top 8", op="logprob", rows=4096, cols=131072, pad=0, type="bf16", top=8, scale=1.0, masked=0.0),
        # the gradient of loss and entropy bonus in policy training; odd sizes
        dict(name="logprob grad 300x10007 f32", op="logprob_grad", rows=300, cols=10007, pad=0, type="f32", scale=1.0, entropy=True, masked=0.0),
        # the gradient of a cross entropy loss on a long batch
        dict(name="logprob grad 8192x32768 bf16", op="logprob_grad", rows=8192, cols=32768, pad=0, type="bf16", scale=1.0, entropy=False, masked=0.0),
        # the weights of a two-layer perceptron 1024 -> 4096 -> 1024, eight of them behind a table of 32768 rows
        dict(name="adamw 100M f32", op="adamw", hidden=1024, layers=8, table=32768, state="f32", param="f32", grad="f32"),
        # a model's weights with 16-bit copies and 16-bit gradients, states in 8 bits
        dict(name="adamw 260M 8 bit", op="adamw", hidden=2048, layers=6, table=32768, state="8bit", param="bf16", grad="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm_grad", "logprob", "logprob_grad", "adamw"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("layernorm", "layernorm_grad"):
        cols = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, max(1, (16384 * 4096 * 2) // (cols * SIZE[kind])))
        return dict(op=op, rows=rows, cols=cols, pad=rng.choice([0, 0, 8, rng.randint(1, 9)]), type=kind,
                    params=rng.choice(["f32", kind]))
    if op in ("logprob", "logprob_grad"):
        cols = _spread(rng, 1000, 200000)
        rows = _spread(rng, 1, min(8192, max(1, (4096 * 32768 * 2) // (cols * SIZE[kind]))))
        c = dict(op=op, rows=rows, cols=cols, pad=rng.choice([0, 0, rng.randint(1, 9)]), type=kind,
                 scale=rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)]), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
        if op == "logprob":
            c["top"] = rng.choice([0, 1, rng.randint(2, 32)])
        else:
            c["entropy"] = rng.choice([True, False])
        return c
    param = rng.choice(["f32", "bf16", "f16"])
    return dict(op=op, hidden=_spread(rng, 16, 1024), layers=rng.randint(1, 12), table=_spread(rng, 100, 32768),
                state=rng.choice(["f32", "8bit"]), param=param, grad=rng.choice(["f32", param]))


def _tensors(case):
    """(elements, weight decay) of the tensors of a model: a table, and for each layer two products' weights and biases
    and a norm's weight and bias, with odd ones among them."""
    h = case["hidden"]
    sizes = [(case["table"] * h, 0.1)]
    for _ in range(case["layers"]):
        sizes += [(h * 4 * h, 0.1), (4 * h, 0.0), (4 * h * h, 0.1), (h, 0.0), (h, 0.0), (h, 0.0)]
    return sizes + [(h * 10, 0.1), (10, 0.0), (1, 0.0)]


def _places(case):
    """(first element, elements, weight decay) of each tensor in the one buffer that holds them all: each begins at a
    multiple of a block."""
    places, at = [], 0
    for n, wd in _tensors(case):
        places.append((at, n, wd))
        at += -(-n // BLOCK) * BLOCK
    return places, at


def work(case):
    op = case["op"]
    if op == "adamw":
        n = sum(s for s, _ in _tensors(case))
        states = 16 if case["state"] == "f32" else 4 + 16 / BLOCK
        copy = SIZE[case["param"]] if case["param"] != "f32" else 0
        return {"bytes": n * (8 + SIZE[case["grad"]] + states + copy), "flops": n * 16}
    rows, cols, t = case["rows"], case["cols"], SIZE[case["type"]]
    if op == "layernorm":
        return {"bytes": 2 * rows * cols * t + 2 * cols * SIZE[case["params"]] + 8 * rows, "flops": 8 * rows * cols}
    if op == "layernorm_grad":
        return {"bytes": 3 * rows * cols * t + 3 * cols * SIZE[case["params"]] + 8 * rows, "flops": 14 * rows * cols}
    if op == "logprob":
        return {"bytes": rows * (cols * t + 8 + 16 + case["top"] * 8), "flops": 7 * rows * cols}
    return {"bytes": rows * (2 * cols * t + 8 + 12 + (8 if case["entropy"] else 0)), "flops": (9 if case["entropy"] else 5) * rows * cols}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _matrix(rows, cols, pad, kind):
    """Rows of `cols` elements that begin cols + pad elements apart."""
    return torch.empty(rows, cols + pad, dtype=kind, device=_device())[:, :cols]


def _logits(case, rnd):
    rows, cols = case["rows"], case["cols"]
    x = _matrix(rows, cols, case["pad"], TYPES[case["type"]])
    x.copy_(torch.randn(rows, cols, generator=rnd, device=x.device, dtype=torch.float32).mul_(2.5))
    tokens = torch.randint(0, cols, (rows,), generator=rnd, device=x.device)
    if case["masked"]:
        # tokens that may not follow; the given token may, but for a row that has none left and one that is not counted
        ruled_out = torch.rand(rows, cols, generator=rnd, device=x.device) < case["masked"]
        ruled_out.scatter_(1, tokens[:, None], False)
        ruled_out[rows // 2] = rows > 1
        x.masked_fill_(ruled_out, -math.inf)
        if rows > 2:
            tokens[rows // 3] = -1
    return x, tokens


def prepare(case, seed):
    rnd = torch.Generator(device=_device())
    rnd.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=rnd, device=_device(), dtype=torch.float32)

    s = {"case": case}
    op = case["op"]
    if op in ("layernorm", "layernorm_grad"):
        rows, cols, kind, params = case["rows"], case["cols"], TYPES[case["type"]], TYPES[case["params"]]
        s["x"] = _matrix(rows, cols, case["pad"], kind)
        s["x"].copy_(normal(rows, cols).mul_(1.5).add_(normal(rows, 1)))
        s["weight"] = normal(cols).mul_(0.2).add_(1).to(params)
        s["eps"] = 1e-5
        if op == "layernorm":
            s["bias"] = normal(cols).mul_(0.2).to(params)
            s["y"] = _matrix(rows, cols, case["pad"], kind)
            s["mean"], s["rstd"] = normal(rows), normal(rows)
        else:
            s["dy"] = _matrix(rows, cols, case["pad"], kind)
            s["dy"].copy_(normal(rows, cols))
            wide = s["x"].double()
            s["mean"] = wide.mean(1).float()
            s["rstd"] = (wide.var(1, unbiased=False) + s["eps"]).rsqrt().float()
            s["dx"] = _matrix(rows, cols, case["pad"], kind)
            s["dweight"], s["dbias"] = torch.empty_like(s["weight"]), torch.empty_like(s["weight"])
    elif op in ("logprob", "logprob_grad"):
        s["x"], s["tokens"] = _logits(case, rnd)
        rows = case["rows"]
        s["stats"], s["entropy"] = normal(rows, 2), normal(rows)
        if op == "logprob":
            s["logprob"] = normal(rows)
            s["top_index"] = torch.empty(rows, case["top"], dtype=torch.int32, device=_device())
            s["top_logprob"] = torch.empty(rows, case["top"], dtype=torch.float32, device=_device())
        else:
            # what the forward pass left: the row's largest logit and the log of its sum, and the entropy
            best, logsum, entropy = _row_sums(s["x"], case["scale"])
            s["stats"] = torch.stack([best, logsum], 1).float()
            s["entropy"] = entropy.float()
            s["dlogprob"] = normal(rows).mul_(0.1).sub_(1.0)
            s["dentropy"] = normal(rows).mul_(0.01).sub_(0.01)
            s["dx"] = _matrix(rows, case["cols"], case["pad"], TYPES[case["type"]])
    else:
        places, n = _places(case)
        here = torch.zeros(n // BLOCK, BLOCK, device=_device(), dtype=torch.bool)
        decay = torch.zeros(n // BLOCK, 1, device=_device())
        for at, count, wd in places:
            here.view(-1)[at:at + count] = True
            decay[at // BLOCK:-(-(at + count) // BLOCK)] = wd
        s["places"], s["decay"] = places, decay
        master = normal(n // BLOCK, BLOCK).mul_(0.05).mul_(here)
        grad = normal(n // BLOCK, BLOCK).mul_(0.01).mul_(normal(n // BLOCK, 1).exp()).mul_(here)
        s["master"], s["grad"] = master, grad.to(TYPES[case["grad"]])
        s["param"] = master.to(TYPES[case["param"]]) if case["param"] != "f32" else None
        m = normal(n // BLOCK, BLOCK).mul_(0.005).mul_(here)
        v = m.square().mul_(2).add_(1e-6).mul_(here)
        if case["state"] == "f32":
            s["m"], s["v"] = m, v
        else:
            # the states as an earlier step left them: 8-bit floats, and for each block what they are multiplied by
            s["m_scale"], s["v_scale"] = m.abs().amax(1) / 448, v.sqrt().amax(1) / 448
            s["m"] = (m / s["m_scale"].clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
            s["v"] = (v.sqrt() / s["v_scale"].clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        s["seed"] = seed % 1000003 + 1
        s["step"] = 100
    return s


def _row_sums(x, scale):
    """Largest logit, log of the sum of exponentials relative to it, and entropy of each row, in 64 bits."""
    best = torch.empty(x.shape[0], dtype=torch.float64, device=x.device)
    logsum, entropy = torch.empty_like(best), torch.empty_like(best)
    step = max(1, (1 << 27) // x.shape[1])
    for a in range(0, x.shape[0], step):
        wide = x[a:a + step].double()
        top = wide.max(1).values
        z = (wide - torch.where(top.isinf(), 0.0, top)[:, None]) * scale
        e = z.exp()
        total = e.sum(1)
        best[a:a + step], logsum[a:a + step] = top, total.log()
        entropy[a:a + step] = torch.where(total > 0, total.log() - (e * z.clamp_min(-1e4)).sum(1) / total.clamp_min(1e-300), 0.0)
    return best, logsum, entropy


# ---- plain forms ------------------------------------------------------------------------------------------------

def _plain_layernorm(s):
    x = s["x"].float()
    mean = x.sum(1) / x.shape[1]
    off = x - mean[:, None]
    rstd = 1 / torch.sqrt((off * off).sum(1) / x.shape[1] + s["eps"])
    y = off * rstd[:, None] * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_layernorm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    n = g.shape[1]
    dx = rstd * (g - g.sum(1, keepdim=True) / n - xh * ((g * xh).sum(1, keepdim=True) / n))
    kind = s["weight"].dtype
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0).to(kind), "dbias": dy.sum(0).to(kind)}


def _plain_logprob(s):
    x, scale, top = s["x"].float(), s["case"]["scale"], s["case"]["top"]
    best = x.amax(1)
    base = torch.where(best.isinf(), torch.zeros_like(best), best)
    z = (x - base[:, None]) * scale
    e = torch.exp(z)
    total = e.sum(1)
    logsum = torch.log(total)
    entropy = torch.where(total > 0, logsum - torch.where(e > 0, e * z, torch.zeros_like(z)).sum(1) / total, torch.zeros_like(total))
    given = s["tokens"].clamp_min(0)[:, None]
    logprob = torch.where(total > 0, torch.gather(z, 1, given)[:, 0] - logsum, torch.full_like(total, -math.inf))
    out = {"logprob": torch.where(s["tokens"] < 0, torch.zeros_like(logprob), logprob),
           "stats": torch.stack([best, logsum], 1), "entropy": entropy}
    if top:
        # whole numbers in the order of the logits, and of the places from the last to the first where these are equal
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
        key = order * (1 << 32) + (MASK32 - torch.arange(x.shape[1], device=x.device))
        index = MASK32 - (torch.topk(key, top, dim=1).values & MASK32)
        out["top_index"] = index.to(torch.int32)
        found = torch.gather(z, 1, index) - logsum[:, None]
        out["top_logprob"] = torch.where(total[:, None] > 0, found, torch.full_like(found, -math.inf))
    return out


def _plain_logprob_grad(s):
    x, scale = s["x"].float(), s["case"]["scale"]
    best, logsum = s["stats"][:, 0], s["stats"][:, 1]
    alive = best > -math.inf
    z = (x - torch.where(alive, best, torch.zeros_like(best))[:, None]) * scale
    logp = z - torch.where(alive, logsum, torch.zeros_like(logsum))[:, None]
    p = torch.exp(logp)
    g = torch.where(alive & (s["tokens"] >= 0), s["dlogprob"], torch.zeros_like(logsum))
    d = -p * g[:, None]
    if s["case"]["entropy"]:
        d -= torch.where(p > 0, p * (logp + s["entropy"][:, None]), torch.zeros_like(p)) * s["dentropy"][:, None]
    d.scatter_add_(1, s["tokens"].clamp_min(0)[:, None], g[:, None])
    return {"dx": (d * scale).to(s["x"].dtype)}


ADAMW = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)


def _random_bits(seed, n, device):
    """32 random bits for each of n elements, from the seed and the element's number (a multiply-xorshift hash)."""
    h = (torch.arange(n, device=device, dtype=torch.int64) * 0x9E3779B1 + seed) & MASK32
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & MASK32
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & MASK32
    return h ^ (h >> 16)


def _to_8_bits(t, rnd):
    """Values of at most 448 in size as 8-bit floats (4 exponent and 3 mantissa bits), rounded up where the 16 random
    bits say so: with a probability of the distance to the lower neighbour."""
    bits = t.abs().view(torch.int32).to(torch.int64)
    normal = (bits + (rnd << 4)) >> 20  # sign 0, exponent with an offset of 127, three bits of mantissa
    small = torch.floor(t.abs() * 512 + rnd.float() * (1 / 65536)).to(torch.int64)  # below 2^-6 in steps of 2^-9
    code = torch.where(t.abs() >= 1 / 64, normal - (120 << 3), small).clamp_max(0x7E)
    return torch.where(t < 0, code | 0x80, code).to(torch.uint8)


def _from_8_bits(code):
    return code.view(torch.float8_e4m3fn).float()


def _plain_adamw(s):
    a = ADAMW
    c1, c2 = 1 - a["beta1"] ** s["step"], 1 - a["beta2"] ** s["step"]
    small = s["case"]["state"] == "8bit"
    g = s["grad"].float()
    if small:
        m = _from_8_bits(s["m"]) * s["m_scale"][:, None]
        r = _from_8_bits(s["v"]) * s["v_scale"][:, None]
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * a["beta1"] + g * (1 - a["beta1"])
    v = v * a["beta2"] + (g * g) * (1 - a["beta2"])
    r = torch.sqrt(v)
    p = s["master"]
    kept = p - p * (s["decay"] * a["lr"])
    p.copy_(kept - (m * (a["lr"] / c1)) / (r * (1 / math.sqrt(c2)) + a["eps"]))
    if s["param"] is not None:
        s["param"].copy_(p)
    if small:
        rnd = _random_bits(s["seed"], g.numel(), g.device).view_as(g)
        s["m_scale"].copy_(m.abs().amax(1) * (1 / 448))
        s["v_scale"].copy_(r.amax(1) * (1 / 448))
        tiny = 2.0 ** -100
        by_m = torch.where(s["m_scale"] > tiny, 1 / s["m_scale"], torch.zeros_like(s["m_scale"]))[:, None]
        by_v = torch.where(s["v_scale"] > tiny, 1 / s["v_scale"], torch.zeros_like(s["v_scale"]))[:, None]
        s["m"].copy_(_to_8_bits((m * by_m).clamp(-448, 448), rnd & 0xFFFF))
        s["v"].copy_(_to_8_bits((r * by_v).clamp_max(448), rnd >> 16))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)


def _adamw_answer(s):
    """The parameters and the states; the 8-bit ones as the numbers that they stand for before their block's scale."""
    out = {"master": s["master"], "m": s["m"], "v": s["v"]}
    if s["param"] is not None:
        out["param"] = s["param"]
    if s["case"]["state"] == "8bit":
        out.update(m_scale=s["m_scale"], v_scale=s["v_scale"], m=s["m"].view(torch.float8_e4m3fn), v=s["v"].view(torch.float8_e4m3fn))
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------

_opened = []


def _framework():
    if not _opened:
        import __graft_entry__
        __graft_entry__.load_package()
        from polarai_framework_amd import capi
        _opened.extend([capi, capi.Device(torch.cuda.current_device())])
    return _opened


def _own(s):
    capi, dev = _framework()
    c, op = s["case"], s["case"]["op"]
    if op == "layernorm":
        dev.flayernorm(s["x"], s["weight"], s["bias"], s["y"], c["rows"], c["cols"], eps=s["eps"], mean=s["mean"], rstd=s["rstd"],
                       dtype=c["type"], param_dtype=c["params"], x_stride=s["x"].stride(0), out_stride=s["y"].stride(0))
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "layernorm_grad":
        dev.flayernorm_grad(s["dy"], s["x"], s["weight"], s["dx"], s["dweight"], s["dbias"], c["rows"], c["cols"], eps=s["eps"],
                            mean=s["mean"], rstd=s["rstd"], dtype=c["type"], param_dtype=c["params"], grad_stride=s["dy"].stride(0),
                            x_stride=s["x"].stride(0), dx_stride=s["dx"].stride(0))
        return {"dx": s["dx"], "dweight": s["dweight"], "dbias": s["dbias"]}
    if op == "logprob":
        dev.flogprob(s["x"], s["tokens"], s["logprob"], c["rows"], c["cols"], scale=c["scale"], stats=s["stats"], entropy=s["entropy"],
                     top=c["top"], top_index=s["top_index"], top_logprob=s["top_logprob"], dtype=c["type"], token_dtype="i64",
                     stride=s["x"].stride(0))
        out = {"logprob": s["logprob"], "stats": s["stats"], "entropy": s["entropy"]}
        if c["top"]:
            out.update(top_index=s["top_index"], top_logprob=s["top_logprob"])
        return out
    if op == "logprob_grad":
        dev.flogprob_grad(s["x"], s["tokens"], s["stats"], s["dlogprob"], s["dx"], c["rows"], c["cols"], scale=c["scale"],
                          entropy=s["entropy"] if c["entropy"] else None, dentropy=s["dentropy"] if c["entropy"] else None,
                          dtype=c["type"], token_dtype="i64", stride=s["x"].stride(0), dlogits_stride=s["dx"].stride(0))
        return {"dx": s["dx"]}
    if "plan" not in s:
        # the list of its tensors that an optimizer keeps
        s["plan"] = capi.adamw_tensors([
            dict(count=n, first=at, weight_decay=wd, grad=s["grad"].view(-1)[at:], param=(s["master"] if s["param"] is None else s["param"]).view(-1)[at:],
                 master=None if s["param"] is None else s["master"].view(-1)[at:], m=s["m"].view(-1)[at:], v=s["v"].view(-1)[at:],
                 m_scale=s["m_scale"][at // BLOCK:] if "m_scale" in s else None, v_scale=s["v_scale"][at // BLOCK:] if "v_scale" in s else None)
            for at, n, wd in s["places"]])
    dev.fadamw(s["plan"], step=s["step"], seed=s["seed"], dtype=c["param"], grad_dtype=c["grad"], state_dtype=c["state"], **ADAMW)
    return None


def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        if own:
            _own(state)
        else:
            _plain_adamw(state)
        return _adamw_answer(state)
    if own:
        return _own(state)
    return {"layernorm": _plain_layernorm, "layernorm_grad": _plain_layernorm_grad, "logprob": _plain_logprob,
            "logprob_grad": _plain_logprob_grad}[op](state)


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------

def _exact_layernorm(s):
    wide = s["x"].double()
    var, mean = torch.var_mean(wide, 1, unbiased=False)
    wide = (wide - mean[:, None]) / torch.sqrt(var + s["eps"])[:, None]
    return {"y": wide * s["weight"].double() + s["bias"].double(), "mean": mean, "rstd": (var + s["eps"]) ** -0.5}


def _exact_layernorm_grad(s):
    dy, r = s["dy"].double(), s["rstd"].double()[:, None]
    centred = s["x"].double() - s["mean"].double()[:, None]
    dweight = torch.mv((dy * centred).t(), r[:, 0])
    g = dy * s["weight"].double()
    along = (g * centred).mean(1, keepdim=True) * r * r
    return {"dx": (g - g.mean(1, keepdim=True) - centred * along) * r, "dweight": dweight, "dbias": dy.sum(0)}


def _exact_logprob(s):
    x, c = s["x"], s["case"]
    best, logsum, entropy = _row_sums(x, c["scale"])
    counted = s["tokens"] >= 0
    given = x[torch.arange(x.shape[0], device=x.device), s["tokens"].clamp_min(0)].double()

    def of(v):
        return torch.where(v.isinf(), -math.inf, (v - best.view(-1, *[1] * (v.dim() - 1))) * c["scale"] - logsum.view(-1, *[1] * (v.dim() - 1)))

    out = {"logprob": torch.where(counted, of(given), 0.0), "stats": torch.stack([best, logsum], 1), "entropy": entropy}
    if c["top"]:
        out["top_index"] = None  # whole numbers have no error
        out["top_logprob"] = of(torch.topk(x.float(), c["top"], dim=1).values.double())
    return out


def _exact_logprob_grad(s):
    x, c = s["x"], s["case"]
    dx = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 27) // x.shape[1])
    for a in range(0, x.shape[0], step):
        rows = slice(a, min(a + step, x.shape[0]))
        best, logsum = s["stats"][rows].double().unbind(1)
        live = ~best.isinf()
        logp = (x[rows].double() - torch.where(live, best, 0.0)[:, None]) * c["scale"] - torch.where(live, logsum, 0.0)[:, None]
        p = logp.exp()
        tokens = s["tokens"][rows]
        hot = (torch.arange(x.shape[1], device=x.device) == tokens[:, None]).double()
        d = (hot - p) * (s["dlogprob"][rows].double() * (live & (tokens >= 0)))[:, None]
        if c["entropy"]:
            d = d - s["dentropy"][rows].double()[:, None] * p * (logp.clamp_min(-1e4) + s["entropy"][rows].double()[:, None])
        dx[rows] = d * c["scale"]
    return {"dx": dx}


def _exact_adamw(s):
    a, small = ADAMW, s["case"]["state"] == "8bit"
    m, v = s["m"], s["v"]
    if small:
        m = m.view(torch.float8_e4m3fn).double() * s["m_scale"].double()[:, None]
        v = (v.view(torch.float8_e4m3fn).double() * s["v_scale"].double()[:, None]) ** 2
    g = s["grad"].double()
    m = m.double().lerp(g, 1 - a["beta1"])
    v = v.double() * a["beta2"] + g ** 2 * (1 - a["beta2"])
    by = a["lr"] / ((v / (1 - a["beta2"] ** s["step"])).sqrt() + a["eps"])
    p = s["master"].double() * (1 - a["lr"] * s["decay"].double()) - by * m / (1 - a["beta1"] ** s["step"])
    out = {"master": p, "m": m, "v": v}
    if s["param"] is not None:
        out["param"] = p
    if small:
        bits = _random_bits(s["seed"], g.numel(), g.device).view_as(g)

        def held(t, rnd):
            # between two neighbouring 8-bit floats, the upper one where distance and random number add up to a step
            scale = t.abs().amax(1, keepdim=True) / 448
            t = t / scale.clamp_min(1e-30)
            step = torch.exp2(torch.frexp(t.abs().clamp_min(2.0 ** -6)).exponent.double() - 4)
            return (torch.floor(t.abs() / step + rnd / 65536) * step).clamp_max(448) * t.sign(), scale[:, 0]

        out["m"], out["m_scale"] = held(m, (bits & 0xFFFF).double())
        out["v"], out["v_scale"] = held(v.sqrt(), (bits >> 16).double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"layernorm": _exact_layernorm, "layernorm_grad": _exact_layernorm_grad, "logprob": _exact_logprob,
            "logprob_grad": _exact_logprob_grad, "adamw": _exact_adamw}[case["op"]](s)
