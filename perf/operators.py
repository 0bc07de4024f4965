"""Measured cases of the 8-bit operators: block quantization, the block-scaled e4m3 product, and the derivative form of an
activation kept as an 8-bit checkpoint.

An 8-bit tensor of shape [rows, cols] is e4m3 values q (row pitch: cols rounded up to 16 bytes) and one f32 scale, a power
of two, per block of 128: "rows" 1 x 128 (scales [ceil(cols/128), rows]), "cols" 128 x 1 ([ceil(rows/128), cols]) or
"tiles" 128 x 128 ([ceil(rows/128), ceil(cols/128)]).  The value it stands for is q * scale, exact in f32.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0


def _ceil(a, b):
    return -(-a // b)


def _pitch(cols):
    return _ceil(cols, 16) * 16


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's activations on their way into a product: latency
        dict(name="quantize_token", op="quantize", rows=1, cols=1024, forms="rows"),
        # the hidden activation of the perceptron configuration, both forms from one read: the forward operand of the next
        # layer and the checkpoint that its weight gradient reads
        dict(name="quantize_hidden", op="quantize", rows=4096, cols=4096, forms="rows+cols"),
        # a weight matrix into 128 x 128 tiles, sizes that end inside a block
        dict(name="quantize_weight_odd", op="quantize", rows=5001, cols=2377, forms="tiles"),
        # serving a single token through the first layer: the weights' bytes bound it
        dict(name="product_token", op="product", m=1, n=4096, k=1024, ta=0, tb=0, fa="rows", fb="tiles", bias=1, act="tanh"),
        # a small serving batch through a square layer of the sweep's largest weights
        dict(name="product_batch32", op="product", m=32, n=8192, k=8192, ta=0, tb=0, fa="rows", fb="tiles", bias=1, act="relu"),
        # the perceptron's first layer, forward: X W1 with bias and activation in the epilogue
        dict(name="product_layer", op="product", m=4096, n=4096, k=1024, ta=0, tb=0, fa="rows", fb="tiles", bias=1, act="tanh"),
        # its weight gradient H^T dZ: both operands stored with the contraction index as the row, a scale per column
        dict(name="product_weight_grad", op="product", m=4096, n=1024, k=4096, ta=1, tb=0, fa="cols", fb="cols", bias=0, act="identity"),
        # input gradient dZ W^T at sizes that end inside blocks, tiles and 16-byte words
        dict(name="product_input_grad_odd", op="product", m=1531, n=2049, k=777, ta=0, tb=1, fa="rows", fb="tiles", bias=0, act="identity"),
        # the sweep's headline product
        dict(name="product_8192", op="product", m=8192, n=8192, k=8192, ta=0, tb=0, fa="rows", fb="tiles", bias=0, act="identity"),
        # derivative form from a small batch's checkpoint: latency
        dict(name="checkpoint_small", op="checkpoint", rows=64, cols=1024, act="tanh", dz=0, forms="rows+cols", db=1),
        # the hidden layer's: everything the rest of the backward pass needs, and dZ itself never stored in 32 bits
        dict(name="checkpoint_hidden", op="checkpoint", rows=4096, cols=4096, act="tanh", dz=0, forms="rows+cols", db=1),
        # dZ in 32 bits from an odd-sized checkpoint of a sigmoid layer, for a backward pass whose products stay in f32
        dict(name="checkpoint_odd", op="checkpoint", rows=6007, cols=1283, act="sigmoid", dz=1, forms="", db=1),
    ]


def _spread(rng, lo, hi):
    """Log-uniform over [lo, hi]; a third of the sizes are multiples of 128, the rest anything."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.34:
        v = max(BLOCK, v // BLOCK * BLOCK)
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "checkpoint"])
    if op == "product":
        while True:
            m, n, k = _spread(rng, 1, 8192), _spread(rng, 16, 8192), _spread(rng, 16, 8192)
            ta, tb = rng.choice([(0, 0), (0, 0), (0, 1), (1, 0), (1, 1)])
            if m * n * k <= 8192 ** 3:
                break
        fa = rng.choice(["cols" if ta else "rows", "cols" if ta else "rows", "tiles"])
        fb = rng.choice(["rows" if tb else "cols", "tiles", "tiles"])
        return dict(op=op, m=m, n=n, k=k, ta=ta, tb=tb, fa=fa, fb=fb, bias=rng.randint(0, 1),
                    act=rng.choice(["identity", "relu", "sigmoid", "tanh"]))
    while True:
        rows, cols = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
        if rows * cols <= 4096 * 4096:
            break
    if op == "quantize":
        return dict(op=op, rows=rows, cols=cols, forms=rng.choice(["rows", "cols", "tiles", "rows+cols"]))
    forms = rng.choice(["", "rows", "cols", "rows+cols"])
    return dict(op=op, rows=rows, cols=cols, act=rng.choice(["tanh", "sigmoid", "relu"]),
                dz=1 if not forms else rng.randint(0, 1), forms=forms, db=rng.randint(0, 1))


def _scale_shape(form, rows, cols):
    rb, cb = _ceil(rows, BLOCK), _ceil(cols, BLOCK)
    return {"rows": (cb, rows), "cols": (rb, cols), "tiles": (rb, cb)}[form]


def _scales(form, rows, cols):
    a, b = _scale_shape(form, rows, cols)
    return a * b


def work(case):
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        ar, ac = (k, m) if case["ta"] else (m, k)
        br, bc = (n, k) if case["tb"] else (k, n)
        b = m * k + k * n + 4 * (_scales(case["fa"], ar, ac) + _scales(case["fb"], br, bc)) + 4 * m * n + 4 * n * case["bias"]
        return {"bytes": b, "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    forms = [f for f in case["forms"].split("+") if f]
    b = 4 * rows * cols + sum(rows * cols + 4 * _scales(f, rows, cols) for f in forms)
    if case["op"] == "checkpoint":
        b += rows * cols + 4 * _scales("cols", rows, cols) + 4 * rows * cols * case["dz"] + 4 * cols * case["db"]
    return {"bytes": b, "flops": 4 * rows * cols * max(1, len(forms))}


# ---- plain forms -------------------------------------------------------------------------------------------------
def _padded(x, br, bc):
    r, c = x.shape
    return torch.nn.functional.pad(x, (0, _ceil(c, bc) * bc - c, 0, _ceil(r, br) * br - r))


def _spread_scales(form, s, rows, cols):
    """The scale of every element, [rows, cols]."""
    if form == "rows":
        return s.t().repeat_interleave(BLOCK, 1)[:, :cols]
    if form == "cols":
        return s.repeat_interleave(BLOCK, 0)[:rows]
    return s.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _quantize(x, form):
    """(q, scales): s = 2^ceil(log2(amax / 448)) over a block's finite values, q = x / s rounded to e4m3."""
    rows, cols = x.shape
    finite = torch.isfinite(x)
    a = torch.where(finite, x.abs(), torch.zeros_like(x))
    br, bc = {"rows": (1, BLOCK), "cols": (BLOCK, 1), "tiles": (BLOCK, BLOCK)}[form]
    p = _padded(a, br, bc)
    amax = p.view(p.shape[0] // br, br, p.shape[1] // bc, bc).amax(dim=(1, 3))
    f, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (f > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(-126, 120)
    s = torch.ldexp(torch.ones_like(amax), e)
    if form == "rows":
        s = s.t().contiguous()
    v = torch.where(finite, x / _spread_scales(form, s, rows, cols), torch.full_like(x, math.nan))
    q = torch.zeros(rows, _pitch(cols), dtype=torch.float8_e4m3fn, device=x.device)
    q[:, :cols] = v.to(torch.float8_e4m3fn)
    return q, s


def _value(q, s, form, rows, cols):
    return q[:, :cols].float() * _spread_scales(form, s, rows, cols)


def _activate(x, act):
    if act == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    return torch.tanh(x) if act == "tanh" else x


def _derivative(y, act):
    if act == "tanh":
        return 1.0 - y * y
    if act == "sigmoid":
        return y * (1.0 - y)
    return (y > 0).to(y.dtype)


# ---- state -------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": dict(case)}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        ar, ac = (k, m) if case["ta"] else (m, k)
        br, bc = (n, k) if case["tb"] else (k, n)
        # activations or gradients with a spread of magnitudes from row to row, weights as an initialiser draws them
        a = _normal(gen, ar, ac) * torch.exp2(torch.randint(-6, 3, (ar, 1), generator=gen, device="cuda").float())
        lim = math.sqrt(6.0 / (n + k))
        b = (torch.rand(br, bc, generator=gen, device="cuda") * 2 - 1) * lim
        st["a"], st["b"] = _quantize(a, case["fa"]), _quantize(b, case["fb"])
        st["bias"] = _normal(gen, n) * 0.1 if case["bias"] else None
        st["c"] = torch.empty(m, n, device="cuda")
    else:
        rows, cols = case["rows"], case["cols"]
        if case["op"] == "quantize":
            # outlier channels beside ordinary ones, as activations have
            st["x"] = _normal(gen, rows, cols) * torch.exp2(torch.randint(-3, 4, (1, cols), generator=gen, device="cuda").float())
        else:
            z = _normal(gen, rows, cols)
            st["y"] = _quantize(_activate(z, case["act"]), "cols")
            # gradients of a mean loss: small, and smaller still for samples that are already right
            st["x"] = _normal(gen, rows, cols) * torch.exp2(torch.randint(-24, -12, (rows, 1), generator=gen, device="cuda").float())
            st["dz"] = torch.empty(rows, cols, device="cuda") if case["dz"] else None
            st["db"] = torch.empty(cols, device="cuda") if case["db"] else None
        st["out"] = {f: (torch.zeros(rows, _pitch(cols), dtype=torch.float8_e4m3fn, device="cuda"),
                         torch.empty(*_scale_shape(f, rows, cols), device="cuda")) for f in case["forms"].split("+") if f}
    if own:
        st["own"] = _handles(st)
    return st


def _handles(st):
    """The framework's tensors over the state's memory, which a user's program holds from call to call."""
    from cleave_b200 import linalg
    case = st["case"]

    def dense(t):
        return None if t is None else linalg.Tensor.from_device_ptr(t.data_ptr(), *t.shape)

    def blocked(qs, form, rows, cols):
        return linalg.QTensor.from_device_ptr(qs[0].data_ptr(), qs[1].data_ptr(), rows, cols, form)

    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"a": blocked(st["a"], case["fa"], *((k, m) if case["ta"] else (m, k))),
                "b": blocked(st["b"], case["fb"], *((n, k) if case["tb"] else (k, n))),
                "bias": dense(st["bias"]), "c": dense(st["c"])}
    rows, cols = case["rows"], case["cols"]
    h = {"x": dense(st["x"]), "out": {f: blocked(qs, f, rows, cols) for f, qs in st["out"].items()}}
    if case["op"] == "checkpoint":
        h.update(y=blocked(st["y"], "cols", rows, cols), dz=dense(st["dz"]), db=dense(st["db"]))
    return h


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _answer(case, out, dz=None, db=None):
    """Quantized forms as e4m3 values without their padding, and scales; dz and db where they are asked for."""
    got = {f: {"q": q[:, :case["cols"]], "s": s} for f, (q, s) in out.items()}
    if dz is not None:
        got["dz"] = dz
    if db is not None:
        got["db"] = db
    return got


def _run_own(st):
    from cleave_b200 import linalg, nn
    case, h = st["case"], st["own"]
    if case["op"] == "product":
        linalg.gemm_q_into(h["c"], h["a"], h["b"], trans_a=bool(case["ta"]), trans_b=bool(case["tb"]), bias=h["bias"],
                           act=case["act"])
        return {"c": st["c"]}
    if case["op"] == "quantize":
        linalg.quantize_into(h["x"], *h["out"].values())
        return _answer(case, st["out"])
    nn.act_bwd_q(h["y"], h["x"], case["act"], *h["out"].values(), dz=h["dz"], db=h["db"])
    return _answer(case, st["out"], st["dz"], st["db"])


def _run_plain(st):
    case = st["case"]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _value(*st["a"], case["fa"], *((k, m) if case["ta"] else (m, k)))
        b = _value(*st["b"], case["fb"], *((n, k) if case["tb"] else (k, n)))
        c = torch.matmul(a.t() if case["ta"] else a, b.t() if case["tb"] else b)
        if st["bias"] is not None:
            c = c + st["bias"]
        return {"c": _activate(c, case["act"])}
    forms = [f for f in case["forms"].split("+") if f]
    if case["op"] == "quantize":
        return _answer(case, {f: _quantize(st["x"], f) for f in forms})
    y = _value(*st["y"], "cols", case["rows"], case["cols"])
    dz = _derivative(y, case["act"]) * st["x"]
    # 64 bits for the column sums: thousands of terms that cancel
    db = dz.double().sum(0).float() if case["db"] else None
    return _answer(case, {f: _quantize(dz, f) for f in forms}, dz if case["dz"] else None, db)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _exact_grid(x, form):
    """Block maxima and the e4m3 grid worked out in 64 bits: the largest power-of-two step count, then round half to even."""
    rows, cols = x.shape
    q = torch.empty_like(x)
    h, w = {"rows": (1, BLOCK), "cols": (BLOCK, 1), "tiles": (BLOCK, BLOCK)}[form]
    big = torch.zeros(_ceil(rows, h), _ceil(cols, w), dtype=torch.float64, device=x.device)
    if h == 1:
        for j in range(big.shape[1]):
            big[:, j] = x[:, j * w:(j + 1) * w].abs().amax(1)
    elif w == 1:
        for i in range(big.shape[0]):
            big[i] = x[i * h:(i + 1) * h].abs().amax(0)
    else:
        for i in range(big.shape[0]):
            strip = x[i * h:(i + 1) * h].abs().amax(0)
            for j in range(big.shape[1]):
                big[i, j] = strip[j * w:(j + 1) * w].amax()
    e = torch.ceil(torch.log2(torch.where(big > 0, big, torch.ones_like(big)) / E4M3_MAX))
    # log2 of a quotient next to a power of two may round across it: settle it by the definition, amax <= 448 * 2^e
    e = torch.where(big > E4M3_MAX * torch.exp2(e), e + 1, e)
    e = torch.where(big <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)
    s = torch.exp2(torch.where(big > 0, e, torch.full_like(e, -126.0)).clamp(-126, 120))
    each = s[torch.arange(rows, device=x.device)[:, None] // h, torch.arange(cols, device=x.device)[None, :] // w]
    v = x / each
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.round(v / step) * step
    return q, (s.t().contiguous() if form == "rows" else s)


def _exact_value(qs, form, rows, cols):
    q, s = qs[0][:, :cols].double(), qs[1].double()
    s = s.t() if form == "rows" else s
    i = torch.arange(rows, device=q.device)[:, None]
    j = torch.arange(cols, device=q.device)[None, :]
    return q * s[i // (1 if form == "rows" else BLOCK), j // (1 if form == "cols" else BLOCK)]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _exact_value(st["a"], case["fa"], *((k, m) if case["ta"] else (m, k)))
        b = _exact_value(st["b"], case["fb"], *((n, k) if case["tb"] else (k, n)))
        c = torch.einsum(("km" if case["ta"] else "mk") + "," + ("nk" if case["tb"] else "kn") + "->mn", a, b)
        if st["bias"] is not None:
            c += st["bias"].double()
        if case["act"] == "relu":
            c = c.clamp_min(0)
        elif case["act"] == "sigmoid":
            c = torch.sigmoid(c)
        elif case["act"] == "tanh":
            c = torch.expm1(2 * c.clamp(-20, 20)) / (torch.expm1(2 * c.clamp(-20, 20)) + 2)
        return {"c": c}
    forms = [f for f in case["forms"].split("+") if f]
    x = st["x"].double()
    if case["op"] == "quantize":
        return {f: dict(zip(("q", "s"), _exact_grid(x, f))) for f in forms}
    y = _exact_value(st["y"], "cols", case["rows"], case["cols"])
    slope = {"tanh": lambda: (1 - y) * (1 + y), "sigmoid": lambda: y - y * y, "relu": lambda: (y > 0).double()}[case["act"]]()
    dz = slope * x
    # A block's scale is a step function of values that carry a rounding of their own, so it has no 64-bit value to be near
    # to; the e4m3 values are within half a step of it wherever the scales agree.
    got = {f: {"q": _exact_grid(dz, f)[0], "s": None} for f in forms}
    if case["dz"]:
        got["dz"] = dz
    if case["db"]:
        got["db"] = dz.sum(0)
    return got
