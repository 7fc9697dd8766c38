"""The int8 operators (int_model_approximation_b200.int8) as measured calls.

Kinds of case:
  product       int8 codes and scales in hand -> the exact int32 product and the rescaled output
  linear        a serving linear: activations in, weight codes laid out once
  linear_train  a training linear: forward and the gradients of activations, weight and bias
                (the weight is quantised in the call, gradients pass straight through the rounding)
  gated         act(x Wg^T + bg) * (x Wu^T + bu), weight codes laid out once
  gated_train   its forward and the gradients of activations and both weights
  gated_tune    forward and the gradients of activations and biases, weight codes frozen
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(name, kind, m, n, k, dtype="bf16", bias=False, act="silu"):
    return {"name": name, "kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "act": act}


def listed():
    return [
        # one token through the gate projection of the 0.5B shapes: latency
        _case("linear_token", "linear", 1, 4864, 896),
        # a decode batch through the down projection of the 7B shapes: weight bandwidth
        _case("linear_decode", "linear", 16, 3584, 18944, bias=True),
        # a ragged batch and odd sizes, nothing a multiple of a tile or of 16 bytes
        _case("linear_ragged", "linear", 77, 333, 1001, "fp16", bias=True),
        # the checkable product of the 0.5B down projection at 512 tokens: int32 sums returned
        _case("product", "product", 512, 896, 4864),
        # a long prompt through the gate projection of the 7B shapes: tensor-core rate
        _case("linear_prefill", "linear", 16384, 18944, 3584),
        # a training step of the 0.5B down projection
        _case("linear_train", "linear_train", 4096, 896, 4864),
        # a small fp32 training step at odd sizes
        _case("linear_train_fp32", "linear_train", 300, 517, 1283, "fp32", bias=True),
        # one token through gate and up of the 7B shapes: weight bandwidth
        _case("gated_token", "gated", 1, 18944, 3584),
        # a decode batch of the 0.5B shapes
        _case("gated_batch", "gated", 45, 4864, 896, "fp16", bias=True, act="gelu"),
        # a long prompt through gate and up of the 7B shapes
        _case("gated_prefill", "gated", 16384, 18944, 3584),
        # a training step of gate and up of the 7B shapes
        _case("gated_train", "gated_train", 4096, 18944, 3584),
        # tuning what lies before a frozen block of the 0.5B shapes
        _case("gated_tune", "gated_tune", 512, 4864, 896, bias=True, act="gelu_tanh"),
    ]


_FACTOR = {"product": 2, "linear": 2, "linear_train": 6, "gated": 4, "gated_train": 12, "gated_tune": 8}


def draw(rng):
    largest = 4.0 * 16384 * 18944 * 3584
    kind = rng.choice(sorted(_FACTOR))
    while True:
        m = int(round(math.exp(rng.uniform(0.0, math.log(16384)))))
        n = int(round(math.exp(rng.uniform(math.log(64), math.log(18944)))))
        k = int(round(math.exp(rng.uniform(math.log(64), math.log(18944)))))
        if rng.random() < 0.5:      # model widths are multiples of 64 as often as not
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        if _FACTOR[kind] * float(m) * n * k <= 0.5 * largest and n * k <= 18944 * 3584:
            break
    return {"kind": kind, "m": m, "n": n, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "bias": rng.random() < 0.5, "act": rng.choice(["silu", "gelu", "gelu_tanh"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(m, k, g, dev):
    """Heavy-tailed activations: Student-t with four degrees of freedom, times 0.5."""
    z = torch.randn((m, k), generator=g, device=dev)
    u = torch.rand((m, k), generator=g, device=dev).clamp_min_(1e-30)
    u.mul_(torch.rand((m, k), generator=g, device=dev).clamp_min_(1e-30))
    return z.div_(u.log_().mul_(-0.5).sqrt_()).mul_(0.5)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    m, n, k, kind = case["m"], case["n"], case["k"], case["kind"]
    dt = DTYPES[case["dtype"]]
    train = kind in ("linear_train", "gated_train", "gated_tune")
    st = {"kind": kind, "act": case["act"], "dtype": dt}
    x = _activations(m, k, g, dev).to(dt)
    names = ["w"] if not kind.startswith("gated") else ["gate", "up"]
    for nm in names:
        w = (torch.randn((n, k), generator=g, device=dev) * 0.02).to(dt)
        if kind in ("linear_train", "gated_train"):
            st[nm] = w
        else:                                   # frozen codes, quantised once per output channel
            st[nm + "_codes"], st[nm + "_scale"] = _quantise(w)
        st[nm + "_bias"] = (torch.randn((n,), generator=g, device=dev) * 0.1).to(dt) if case["bias"] else None
    if kind == "product":
        st["x_codes"], st["x_scale"] = _quantise(x)
    else:
        st["x"] = x
    if train:
        # gradients whose size differs from token to token
        size = torch.exp(torch.randn((m, 1), generator=g, device=dev)) * 1e-2
        st["dy"] = (torch.randn((m, n), generator=g, device=dev) * size).to(dt)
    if own:
        from int_model_approximation_b200 import int8

        for nm in names:
            if nm + "_codes" in st and kind != "product":
                st[nm + "_weight"] = int8.Int8Weight(st[nm + "_codes"], st[nm + "_scale"])
            if train:
                for t in (st.get(nm), st[nm + "_bias"]):
                    if t is not None:
                        t.requires_grad_()
        if train:
            st["x"].requires_grad_()
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantise(x):
    """int8 codes of each row and its fp32 scale, amax / 127."""
    x = x.float()
    amax = x.abs().amax(dim=1, keepdim=True)
    scale = (amax / torch.full_like(amax, 127.0)).clamp_min(1e-12)
    return (x / scale).round().clamp(-127, 127).to(torch.int8), scale


def _product(a, b):
    """The exact int32 product of int8 rows: pieces of 1024 columns are exact in 32-bit floats."""
    out = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.int32, device=a.device)
    for k0 in range(0, a.shape[1], 1024):
        out += (a[:, k0:k0 + 1024].float() @ b[:, k0:k0 + 1024].float().t()).to(torch.int32)
    return out


def _rescaled(c, x_scale, w_scale, bias):
    y = c.float().mul_(x_scale).mul_(w_scale.reshape(1, -1))
    return y if bias is None else y.add_(bias.float())


def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain(st):
    dt, kind = st["dtype"], st["kind"]
    if kind == "product":
        c = _product(st["x_codes"], st["w_codes"])
        return {"c": c, "y": _rescaled(c, st["x_scale"], st["w_scale"], st["w_bias"]).to(dt)}
    q, s = _quantise(st["x"])
    names = ["gate", "up"] if kind.startswith("gated") else ["w"]
    codes, scales, raw = [], [], []
    for nm in names:
        wq, ws = (st[nm + "_codes"], st[nm + "_scale"]) if nm + "_codes" in st else _quantise(st[nm])
        codes.append(wq)
        scales.append(ws.reshape(1, -1))
        raw.append(_rescaled(_product(q, wq), s, ws, st[nm + "_bias"]))
    out = {}
    if kind.startswith("gated"):
        a, da = _act(raw[0], st["act"])
        out["h"] = (a * raw[1]).to(dt)
        if kind != "gated":
            dh = st["dy"].float()
            d = [dh * raw[1] * da, dh * a]
    else:
        out["y"] = raw[0].to(dt)
        if kind == "linear_train":
            d = [st["dy"].float()]
    if "dy" in st:
        out["dx"] = sum((di * sc) @ wq.float() for di, sc, wq in zip(d, scales, codes)).to(dt)
        for nm, di in zip(names, d):
            if nm in st:
                out["d" + nm] = (di.t() @ (q.float() * s)).to(dt)
            if st[nm + "_bias"] is not None:
                out["d" + nm + "_bias"] = di.double().sum(dim=0).to(dt)
    return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _calls(st):
    from int_model_approximation_b200 import int8

    dt, kind = st["dtype"], st["kind"]
    if kind == "product":
        c, y = int8.int8_gemm(st["x_codes"], st["w_codes"], want_c=True, x_scale=st["x_scale"], w_scale=st["w_scale"],
                              bias=st["w_bias"], y_dtype=dt)
        return {"c": c, "y": y}
    if kind == "linear":
        return {"y": int8.int8_linear(st["x"], st["w_weight"], st["w_bias"])}
    if kind == "gated":
        return {"h": int8.int8_gated(st["x"], st["gate_weight"], st["up_weight"], st["gate_bias"], st["up_bias"],
                                     activation=st["act"])}
    if kind == "linear_train":
        y = int8.int8_linear(st["x"], st["w"], st["w_bias"])
        out, leaves = {"y": y.detach()}, {"dx": st["x"], "dw": st["w"], "dw_bias": st["w_bias"]}
    else:
        weight = {nm: st[nm] if kind == "gated_train" else st[nm + "_weight"] for nm in ("gate", "up")}
        y = int8.int8_gated(st["x"], weight["gate"], weight["up"], st["gate_bias"], st["up_bias"], activation=st["act"])
        out, leaves = {"h": y.detach()}, {"dx": st["x"]}
        for nm in ("gate", "up"):
            leaves["d" + nm] = st.get(nm)
            leaves["d" + nm + "_bias"] = st[nm + "_bias"]
    leaves = {name: t for name, t in leaves.items() if t is not None}
    out.update(zip(leaves, torch.autograd.grad(y, list(leaves.values()), st["dy"])))
    return out


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _codes64(x):
    """Codes and scale by definition: both quotients rounded to fp32, everything else exact."""
    x = x.detach().double()
    s = torch.clamp_min((x.abs().max(dim=1).values / 127.0).float(), 1e-12).double()
    return torch.clamp(torch.round((x / s[:, None]).float()), -127, 127).double(), s


def exact(case, seed):
    st = prepare(case, seed)
    kind = st["kind"]
    gated = kind.startswith("gated")
    if kind == "product":
        q, s = st["x_codes"].double(), st["x_scale"].double().flatten()
    else:
        q, s = _codes64(st["x"])
    pre = {}
    w_hat = {}
    for nm in (("gate", "up") if gated else ("w",)):
        if nm + "_codes" in st:
            w, t = st[nm + "_codes"].double(), st[nm + "_scale"].double().flatten()
        else:
            w, t = _codes64(st[nm])
        c = torch.mm(q, w.T)
        if kind == "product":
            whole = c.round().to(torch.int32)
        c *= s[:, None]
        c *= t
        if st[nm + "_bias"] is not None:
            c += st[nm + "_bias"].detach().double()
        pre[nm] = c
        w_hat[nm] = w.mul_(t[:, None])
    if kind == "product":
        return {"c": whole, "y": pre["w"]}
    if not gated:
        out = {"y": pre["w"]}
        grad = {"w": st["dy"].double()} if "dy" in st else {}
    else:
        g, u = pre["gate"], pre["up"]
        if st["act"] == "silu":
            value = g * torch.sigmoid(g)
            slope = torch.sigmoid(g) + value * torch.sigmoid(-g)
        elif st["act"] == "gelu":
            value = 0.5 * g * torch.erfc(-g / math.sqrt(2.0))
            slope = 0.5 * torch.erfc(-g / math.sqrt(2.0)) + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        else:
            z = math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
            value = g * torch.sigmoid(2 * z)
            slope = torch.sigmoid(2 * z) + value * torch.sigmoid(-2 * z) * 2 * math.sqrt(2.0 / math.pi) * (
                1 + 0.134145 * g.square())
        out = {"h": value * u}
        grad = {"gate": st["dy"].double() * u * slope, "up": st["dy"].double() * value} if "dy" in st else {}
    if grad:
        dx = 0
        x_hat = q * s[:, None]
        for nm, d in grad.items():
            dx = dx + torch.mm(d, w_hat[nm])
        out["dx"] = dx
        for nm, d in grad.items():
            if nm in st:
                out["d" + nm] = torch.mm(d.T, x_hat)
            if st[nm + "_bias"] is not None:
                out["d" + nm + "_bias"] = d.sum(dim=0)
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    m, n, k, kind = case["m"], case["n"], case["k"], case["kind"]
    e = 4 if case["dtype"] == "fp32" else 2
    pair = 2 if kind.startswith("gated") else 1
    trained = kind in ("linear_train", "gated_train")
    nbytes = m * n * e + pair * n * k * (e if trained else 1)           # output, weights
    nbytes += m * k * (1 if kind == "product" else e)                   # activations or their codes
    if not trained:
        nbytes += pair * n * 4
    if case["bias"]:
        nbytes += pair * n * e
    if kind == "product":
        nbytes += 4 * m * n + 4 * m
    if kind in ("linear_train", "gated_train", "gated_tune"):
        nbytes += m * n * e + m * k * e                                 # dy, dx
        if trained:
            nbytes += pair * n * k * e                                  # weight gradients
        if case["bias"]:
            nbytes += pair * n * e
    return {"bytes": nbytes, "flops": _FACTOR[kind] * m * n * k}
