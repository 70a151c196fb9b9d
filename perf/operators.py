"""The measured operators: layer normalisation forward and backward, the gradient norm over many tensors, and the
AdamW step over many tensors with its state in 32 or in 8 bits.

`run` computes them in their plain form (elementary tensor operations) or, where `own` is true, through the calls a
user makes of this package.  `exact` gives the same outputs from the definitions in 64 bits.

Optimizer arenas: tensor i starts at a multiple of BLOCK elements, the gap behind it holds zeros.  The state is one
buffer: 32 bits: m, v as f32; 8 bits: codes of m (signed), codes of sqrt(v) (unsigned), then one f32 scale per block
of BLOCK elements for each.  Both are companded by a square root: m = s (c / 127)^2 sign(c), sqrt(v) = s (c / 255)^2.
"""
import math

import torch

own = False

BLOCK = 256
TINY = 2.0 ** -100  # the least scale of a block of 8-bit state
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.1
LN_EPS = 1e-5
CLIP_EPS = 1e-6
LARGEST = 16384 * 4096  # elements of the largest normalised activation


def _decoder_lens(layers, width):
    """Parameter counts of `layers` decoder blocks: four square projections, two of the feed-forward, norms, biases."""
    one = [width, width] + [width * width, width] * 4 + [width, width] + [4 * width * width, 4 * width, 4 * width * width, width]
    return " ".join(str(n) for n in one * layers)


def listed():
    return [
        # one row: the normalisation of a single decoded token
        {"name": "norm 1x1024", "op": "norm", "rows": 1, "cols": 1024, "wide": 0, "dtype": "f32"},
        # a batch whose features are a slice of a wider activation, rows 16-byte aligned
        {"name": "norm 8192x1000 of 1024", "op": "norm", "rows": 8192, "cols": 1000, "wide": 24, "dtype": "f32"},
        # odd sizes in double precision, the type gradient checks run in
        {"name": "norm 1237x1001 f64", "op": "norm", "rows": 1237, "cols": 1001, "wide": 0, "dtype": "f64"},
        # the tokens of a long training batch at a wide model
        {"name": "norm 16384x4096", "op": "norm", "rows": 16384, "cols": 4096, "wide": 0, "dtype": "f32"},
        # a small hidden layer's batch
        {"name": "norm grad 128x512", "op": "norm_grad", "rows": 128, "cols": 512, "wide": 0, "dtype": "f32"},
        # an ordinary training batch, rows that are no multiple of a warp's vectors
        {"name": "norm grad 8192x1000", "op": "norm_grad", "rows": 8192, "cols": 1000, "wide": 0, "dtype": "f32"},
        {"name": "norm grad 2049x777 f64", "op": "norm_grad", "rows": 2049, "cols": 777, "wide": 0, "dtype": "f64"},
        {"name": "norm grad 16384x4096", "op": "norm_grad", "rows": 16384, "cols": 4096, "wide": 0, "dtype": "f32"},
        # the six tensors of the 784-512-256-10 classifier, clipped: launch-bound
        {"name": "adamw 32 bits, classifier", "op": "adamw", "bits": 32, "clip": 1.0, "step": 100,
         "lens": "401408 512 131072 256 2560 10"},
        # eight decoder blocks of width 1024, 128 tensors, 0.1 G parameters
        {"name": "adamw 32 bits, decoder", "op": "adamw", "bits": 32, "clip": 0.0, "step": 1000, "lens": _decoder_lens(8, 1024)},
        # the 17 M convolutional network's twelve tensors
        {"name": "adamw 8 bits, wide CNN", "op": "adamw", "bits": 8, "clip": 0.0, "step": 100,
         "lens": "3456 128 128 128 294912 256 256 256 16777216 1024 10240 10"},
        {"name": "adamw 8 bits, decoder", "op": "adamw", "bits": 8, "clip": 1.0, "step": 1000, "lens": _decoder_lens(8, 1024)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "adamw", "adamw", "adamw"])
    if kind != "adamw":
        dtype = rng.choice(["f32", "f32", "f32", "f64"])
        cols = _log_int(rng, 32, 16384)
        rows = _log_int(rng, 1, min(65536, LARGEST // (2 if dtype == "f64" else 1) // cols))
        if rng.random() < 0.4:  # widths of models are mostly multiples of 8
            cols = max(32, cols // 8 * 8)
        return {"op": kind, "rows": rows, "cols": cols, "wide": rng.choice([0, 0, 0, 8, 5]), "dtype": dtype}
    tensors = _log_int(rng, 1, 300)
    total = _log_int(rng, 1000, 100_000_000)
    share = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(tensors)]
    lens = [max(1, int(total * s / sum(share))) for s in share]
    return {"op": "adamw", "bits": rng.choice([32, 8]), "clip": rng.choice([0.0, 1.0]), "step": _log_int(rng, 2, 100_000),
            "lens": " ".join(str(n) for n in lens)}


# ---- inputs ----------------------------------------------------------------------------------------

def _lens(case):
    return [int(n) for n in case["lens"].split()]


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def _no_decay(n):
    """Vectors (biases, gains) are exempt from weight decay; here: every tensor of at most 4096 elements."""
    return n <= 4096


def _inputs_norm(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.float64 if case["dtype"] == "f64" else torch.float32
    rows, cols, wide = case["rows"], case["cols"], case["wide"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=gen)

    # activations: every row with an offset and a spread of its own
    x = normal(rows, cols + wide) * torch.exp(0.5 * normal(rows, 1)) + 0.5 * normal(rows, 1)
    s = {"x": x[:, :cols], "weight": 1 + 0.2 * normal(cols), "bias": 0.1 * normal(cols)}
    if case["op"] == "norm":
        s |= {"y": torch.empty(rows, cols, device="cuda", dtype=dt), "mean": torch.empty(rows, device="cuda", dtype=dt),
              "rstd": torch.empty(rows, device="cuda", dtype=dt)}
    else:
        s["dy"] = normal(rows, cols) * 0.1
        x64 = s["x"].double()
        s["mean"] = x64.mean(1).to(dt)
        s["rstd"] = (x64.var(1, unbiased=False) + LN_EPS).rsqrt().to(dt)
        s |= {"dx": torch.empty(rows, cols, device="cuda", dtype=dt), "dweight": torch.empty(cols, device="cuda", dtype=dt),
              "dbias": torch.empty(cols, device="cuda", dtype=dt)}
    return s


def _inputs_adamw(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lens(case)
    starts, at = [], 0
    for n in lens:
        starts.append(at)
        at += _padded(n)
    blocks = at // BLOCK

    def blank():
        return torch.zeros(at, device="cuda")

    theta, grad, m, v = blank(), blank(), blank(), blank()
    decay = torch.ones(blocks, 1, device="cuda")
    for a, n in zip(starts, lens):
        # a scale per tensor, rows of very different size inside it
        size = 0.02 * math.exp(0.7 * math.sin(a + n))

        def some(k):
            return torch.randn(n, device="cuda", generator=gen) * k

        theta[a:a + n] = some(0.05)
        grad[a:a + n] = some(size) * torch.exp(some(1.0))
        m[a:a + n] = some(0.3 * size) * torch.exp(some(1.0))
        v[a:a + n] = (size * torch.exp(some(1.0))).square()
        if _no_decay(n):
            decay[a // BLOCK:(a + _padded(n)) // BLOCK] = 0
    s = {"theta": theta, "grad": grad, "decay": decay, "lens": lens, "starts": starts, "blocks": blocks}
    if case["bits"] == 32:
        s["state"] = torch.cat([m, v])
        s |= {"m": s["state"][:at], "v": s["state"][at:]}
    else:
        s["state"] = torch.zeros(2 * at + 8 * blocks, device="cuda", dtype=torch.uint8)
        s |= {"mc": s["state"][:at].view(torch.int8), "vc": s["state"][at:2 * at]}
        s |= {"ms": s["state"][2 * at:2 * at + 4 * blocks].view(torch.float32), "vs": s["state"][2 * at + 4 * blocks:].view(torch.float32)}
        _encode(s, m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK))
        s |= {"m": torch.zeros(at, device="cuda"), "v": torch.zeros(at, device="cuda")}
    if case["clip"]:
        s |= {"norm": torch.zeros(1, device="cuda"), "scale": torch.zeros(1, device="cuda")}
    return s


_backends = {}


def _backend():
    """One backend on the current device and stream, kept as a program keeps it."""
    from weta_b200.backend import B200Backend

    at = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if at not in _backends:
        _backends[at] = B200Backend(at[0], stream=at[1])
    return _backends[at]


def prepare(case, seed):
    s = _inputs_adamw(case, seed) if case["op"] == "adamw" else _inputs_norm(case, seed)
    s["case"] = dict(case)
    if own:
        from weta_b200 import layers, optim
        from weta_b200.core import DType, Layout

        be = s["be"] = _backend()
        if case["op"] == "adamw":
            thetas = [be.wrap_pointer(s["theta"].data_ptr() + 4 * a, n, DType.F32) for a, n in zip(s["starts"], s["lens"])]
            grads = [be.wrap_pointer(s["grad"].data_ptr() + 4 * a, n, DType.F32) for a, n in zip(s["starts"], s["lens"])]
            s["opt"] = optim.AdamMulti(be, thetas, state_bits=case["bits"], no_decay=[_no_decay(n) for n in s["lens"]], lr=LR,
                                       betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, decoupled=True,
                                       state=be.wrap_pointer(s["state"].data_ptr(), s["state"].nbytes // 4, DType.F32), keep_state=True)
            s["opt"].set_grads(grads)
            s["own"] = {k: be.wrap_pointer(s[k].data_ptr(), s[k].numel(), DType.F32) for k in ("m", "v", "norm", "scale") if k in s}
        else:
            dt = s["dt"] = DType.F64 if case["dtype"] == "f64" else DType.F32
            s["own"] = {k: be.wrap_pointer(t.data_ptr(), t.numel(), dt) for k, t in s.items() if isinstance(t, torch.Tensor)}
            s["lx"] = Layout([case["rows"], case["cols"]], s["x"].stride(), 0)
            s["ly"] = Layout.contiguous([case["rows"], case["cols"]])
            if case["op"] == "norm_grad":
                s["work"] = layers.layer_norm_workspace(be, case["rows"], case["cols"], dt)
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(s):
    return {"norm": _norm, "norm_grad": _norm_grad, "adamw": _adamw}[s["case"]["op"]](s)


def _norm(s):
    if own:
        from weta_b200 import layers

        o = s["own"]
        layers.layer_norm_fwd(s["be"], o["x"], s["lx"], s["dt"], 1, o["weight"], o["bias"], LN_EPS, out=(o["y"], o["mean"], o["rstd"]))
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    x = s["x"]
    mean = x.sum(1, keepdim=True) / x.shape[1]
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).sum(1, keepdim=True) / x.shape[1] + LN_EPS)
    return {"y": d * rstd * s["weight"] + s["bias"], "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _norm_grad(s):
    if own:
        from weta_b200 import layers

        o = s["own"]
        layers.layer_norm_bwd(s["be"], o["x"], s["lx"], o["dy"], s["ly"], s["dt"], 1, o["weight"], o["mean"], o["rstd"],
                              out=(o["dx"], o["dweight"], o["dbias"]), workspace=s["work"])
        return {"dx": s["dx"], "dweight": s["dweight"], "dbias": s["dbias"]}
    x, dy, n = s["x"], s["dy"], s["x"].shape[1]
    rstd = s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    g = dy * s["weight"]
    dx = rstd * (g - g.sum(1, keepdim=True) / n - xhat * ((g * xhat).sum(1, keepdim=True) / n))
    return {"dx": dx, "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _encode(s, m, root):
    """8-bit state of a [blocks, BLOCK] pair (m, sqrt(v)) into the buffers of `s`."""
    ms = m.abs().amax(1, keepdim=True).clamp(min=TINY)
    vs = root.amax(1, keepdim=True).clamp(min=TINY)
    levels = torch.tensor([127.0 ** 2, 255.0 ** 2], device="cuda")
    mc = torch.round(torch.sqrt(m.abs() * (levels[0] / ms))).clamp(max=127)
    vc = torch.round(torch.sqrt(root * (levels[1] / vs))).clamp(max=255)
    vc = torch.where(root > 0, vc.clamp(min=1), vc)  # what is not zero stays so
    s["mc"].copy_(torch.where(m < 0, -mc, mc).to(torch.int8).view(-1))
    s["vc"].copy_(vc.to(torch.uint8).view(-1))
    s["ms"].copy_(ms[:, 0])
    s["vs"].copy_(vs[:, 0])


def _decode(s):
    """(m, v) as [blocks, BLOCK]."""
    c = s["mc"].float().view(-1, BLOCK)
    m = c * c.abs() * (s["ms"] * (1 / 127.0 ** 2))[:, None]
    r = s["vc"].float().view(-1, BLOCK)
    root = r * r * (s["vs"] * (1 / 255.0 ** 2))[:, None]
    return m, root * root


def _adamw(s):
    case = s["case"]
    if own:
        o = s["own"]
        if case["clip"]:
            s["opt"].grad_norm(case["clip"], out=(o["norm"], o["scale"]))
        s["opt"].step(case["step"], grad_scale=o["scale"] if case["clip"] else None)
        if case["bits"] == 8:
            s["opt"].read_state(out=(o["m"], o["v"]))
    else:
        theta, g = s["theta"].view(-1, BLOCK), s["grad"].view(-1, BLOCK)
        if case["clip"]:
            norm = torch.sqrt(g.double().square().sum())  # a long sum: 64 bits
            s["norm"].copy_(norm)
            s["scale"].copy_((case["clip"] / (norm + CLIP_EPS)).clamp(max=1.0))
            g = g * s["scale"]
        m, v = (s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)) if case["bits"] == 32 else _decode(s)
        th = torch.where(s["decay"] > 0, theta * (1 - LR * DECAY), theta)
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        root = torch.sqrt(v)
        den = root * (1 / math.sqrt(1 - BETA2 ** case["step"])) + EPS
        theta.copy_(th - (m / den) * (LR / (1 - BETA1 ** case["step"])))
        if case["bits"] == 8:
            _encode(s, m, root)
            m, v = _decode(s)
        s["m"].copy_(m.reshape(-1))
        s["v"].copy_(v.reshape(-1))
    return {k: s[k] for k in ("theta", "m", "v", "norm", "scale") if k in s}


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    if case["op"] == "adamw":
        n, b = sum(_lens(case)), case["bits"] // 8
        scales = sum(-(-k // BLOCK) for k in _lens(case)) * 16 if b == 1 else 0
        back = 8 * n if b == 1 else 0  # the 8-bit state, read back as the values it stands for
        return {"bytes": 12 * n + 4 * n * b + scales + back, "flops": (18 if b == 4 else 34) * n + (3 * n if case["clip"] else 0)}
    r, c, b = case["rows"], case["cols"], 8 if case["dtype"] == "f64" else 4
    if case["op"] == "norm":
        return {"bytes": b * (2 * r * c + 2 * c + 2 * r), "flops": 8 * r * c}
    return {"bytes": b * (3 * r * c + 3 * c + 2 * r), "flops": 14 * r * c}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "adamw":
        return _exact_adamw(case, _inputs_adamw(case, seed))
    s = {k: t.double() for k, t in _inputs_norm(case, seed).items()}
    x, c = s["x"], case["cols"]
    if case["op"] == "norm":
        mean = torch.einsum("rc->r", x) / c
        centred = x - mean[:, None]
        deviation = torch.sqrt(torch.einsum("rc,rc->r", centred, centred) / c + LN_EPS)
        return {"y": centred / deviation[:, None] * s["weight"] + s["bias"], "mean": mean, "rstd": deviation.reciprocal()}
    rows = (x - s["mean"][:, None]).mul_(s["rstd"][:, None])
    up = s["dy"] * s["weight"]
    along = torch.einsum("rc,rc->r", up, rows) / c
    level = torch.einsum("rc->r", up) / c
    return {"dx": (up - level[:, None] - along[:, None] * rows) * s["rstd"][:, None],
            "dweight": torch.einsum("rc,rc->c", s["dy"], rows), "dbias": torch.einsum("rc->c", s["dy"])}


def _exact_adamw(case, s):
    # The 8-bit state is defined on values rounded to f32 (a code next to a border goes by them): where it is kept, every
    # step below rounds its 64-bit result to f32, and nowhere else.
    def r(a):
        return a.float().double() if case["bits"] == 8 else a

    def k(a):
        return float(torch.tensor(a, dtype=torch.float32)) if case["bits"] == 8 else a

    wide = {key: t.double() for key, t in s.items() if isinstance(t, torch.Tensor)}
    g, out = wide["grad"], {}
    if case["clip"]:
        total = torch.linalg.vector_norm(g)
        factor = torch.minimum(case["clip"] / (total + CLIP_EPS), torch.ones_like(total))
        out = {"norm": total[None], "scale": factor[None]}
        g = r(g * r(factor))

    def per_element(a):
        return torch.repeat_interleave(a, BLOCK)

    if case["bits"] == 32:
        m, v = wide["m"], wide["v"]
    else:
        m = r(wide["mc"] * wide["mc"].abs() * per_element(r(wide["ms"] * k(1 / 16129))))
        v = r(r(wide["vc"] ** 2 * per_element(r(wide["vs"] * k(1 / 65025)))) ** 2)
    keep = per_element(torch.where(wide["decay"][:, 0] > 0, k(1 - LR * DECAY), 1.0))
    m = r(r(m * k(BETA1)) + r(g * k(1 - BETA1)))
    v = r(r(v * k(BETA2)) + r(r(g * g) * k(1 - BETA2)))
    root = r(v.sqrt())
    den = r(r(root * k(1 / math.sqrt(1 - BETA2 ** case["step"]))) + k(EPS))
    out["theta"] = r(r(wide["theta"] * keep) - r(r(m / den) * k(LR / (1 - BETA1 ** case["step"]))))
    if case["bits"] == 8:
        def stored(a, top):
            """What the codes 0..top stand for; the magnitude alone."""
            most = a.view(-1, BLOCK).amax(1).clamp(min=TINY)
            code = r(r(a * per_element(r(top * top / most))).sqrt()).round().clamp(max=top)
            code = torch.where((a > 0) & (top == 255), code.clamp(min=1), code)
            return r(code * code * per_element(r(most * k(1 / (top * top)))))

        m, v = stored(m.abs(), 127) * m.sign(), r(stored(root, 255) ** 2)
    return out | {"m": m, "v": v}
