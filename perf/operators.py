"""What a training step built on deepfuse_amd has it do around its fp8 Linears, with each operator's plain form.

A case is a dict of plain values; its "kind" says which operator it runs:

  ln_forward     LayerNorm over rows, with the residual add in front of it, keeping the row statistics
  ln_backward    its backward: dx (plus the residual path's gradient), dgamma and dbeta
  adamw          an AdamW step over many tensors, with states in 32 bits or in 8 (e4m3 codes and a scale per 256 values)
  experts_fwd    the products of a Linear's experts with their rows, rows sorted by expert, on fp8 codes
  experts_bwd    the same Linear's dX and dW

Where `own` is false, run() computes in elementary torch operations, in 32 bits; where it is true, it calls the library.
The sizes are those of GPT-2 small and GPT-2 XL blocks, as bench.py and the tests run them, and odd ones.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
FMAX = {E4: 448.0, E5: 57344.0}
BLOCK = 256  # values that share a scale in 8-bit states
EPS = 1e-5  # of the norm
LR, BETA1, BETA2, ADAM_EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1

# one block's parameters: the four Linears' weights and biases, the two norms' gamma and beta
SMALL = "2304x768,2304,768x768,768,768x2304,768,2304x768,2304,768,768,768,768"
XL = "4800x1600,4800,1600x1600,1600,6400x1600,6400,1600x6400,1600,1600,1600,1600,1600"


def ln(name, kind, rows, cols, dtype="bf16", residual=True):
    return {"name": name, "kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "residual": residual}


def adamw(name, shapes, copies=1, state="8", grad="f32", copy="none"):
    return {"name": name, "kind": "adamw", "shapes": shapes, "copies": copies, "state": state, "grad": grad,
            "copy": copy}


def experts(name, kind, rows, count, k, n, skew="even", dtype="bf16"):
    return {"name": name, "kind": kind, "rows": rows, "experts": count, "k": k, "n": n, "skew": skew, "dtype": dtype}


def listed():
    return [
        # one token of a small model being generated: all latency
        ln("ln_forward_token", "ln_forward", 1, 768),
        # a large model's norm over a full batch, the residual stream carried along
        ln("ln_forward_xl", "ln_forward", 16384, 1600),
        # a small model's norm over one short sequence, gradients on a small batch
        ln("ln_backward_small", "ln_backward", 512, 768),
        # a large model's norm over a full batch
        ln("ln_backward_xl", "ln_backward", 16384, 1600),
        # a width that is no multiple of anything, in half precision, no residual path
        ln("ln_backward_ragged", "ln_backward", 1000, 771, dtype="f16", residual=False),
        # one block of a small model, 32-bit states, as Adam runs today
        adamw("adamw32_small", SMALL, state="32"),
        # the same tensors of two large blocks with 8-bit states and 16-bit gradients, the weights' bf16 copies written
        adamw("adamw8_xl_2", XL, copies=2, grad="bf16", copy="bf16"),
        # a norm's parameters alone: the smallest update
        adamw("adamw8_norm", "771,771"),
        # generation: a few tokens, each sent to two of many experts, bound by reading their weights
        experts("experts_fwd_decode", "experts_fwd", 64, 32, 1600, 1600, skew="skewed"),
        # a large model's fc1 over a full batch, eight experts
        experts("experts_fwd_xl", "experts_fwd", 16384, 8, 1600, 6400),
        # its backward
        experts("experts_bwd_xl", "experts_bwd", 16384, 8, 1600, 6400),
        # a layer of odd sizes with uneven experts, some of them without a row, in half precision
        experts("experts_bwd_ragged", "experts_bwd", 1000, 12, 771, 1037, skew="skewed", dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: any number, or, as most models have them, a multiple of 64."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.4 else min(hi, max(64, (w + 32) // 64 * 64))


MOST = {"bytes": 1.2e9, "flops": 6.7e11}  # a drawn case stays below the largest listed ones


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if all(w[k] <= MOST[k] for k in MOST):
            return c


def _draw(rng):
    kind = rng.choice(["ln_forward", "ln_backward", "ln_backward", "adamw", "adamw", "experts_fwd", "experts_bwd"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind.startswith("ln"):
        c = ln("", kind, _log(rng, 1, 16384), _width(rng, 32, 6400), dtype, rng.random() < 0.6)
    elif kind == "adamw":
        shapes = []
        for _ in range(_log(rng, 1, 24)):
            n = _width(rng, 64, 6400)
            shapes.append("%d" % n if rng.random() < 0.5 else "%dx%d" % (n, _width(rng, 64, 1600)))
        c = adamw("", ",".join(shapes), rng.choice([1, 1, 2]), rng.choice(["8", "8", "32"]),
                  rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice(["none", "bf16", "f16"]))
    else:
        c = experts("", kind, _log(rng, 1, 16384), _log(rng, 1, 64), _width(rng, 64, 6400), _width(rng, 64, 6400),
                    rng.choice(["even", "skewed"]), dtype)
    del c["name"]
    return c


# ---- sizes, inputs ---------------------------------------------------------------------------------------------------

def _sizes(case):
    return [math.prod(int(v) for v in s.split("x")) for s in case["shapes"].split(",")] * case["copies"]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _codes(x, fmt):
    """fp8 codes of x at its per-tensor scale, rows padded to a multiple of 16 with zero codes, and the scale."""
    s = (x.abs().max() / FMAX[fmt]).reshape(1)
    q = (x / s).clamp(-FMAX[fmt], FMAX[fmt]).to(fmt).view(torch.uint8)
    return torch.nn.functional.pad(q, (0, -q.shape[-1] % 16)).contiguous(), s


def _bounds(case, seed):
    """First row of each expert: "even" as a balanced router leaves them, "skewed" with a few busy and some idle ones."""
    g = torch.Generator().manual_seed(int(seed))
    p = torch.rand(case["experts"], generator=g) * 0.4 + 0.8
    if case["skew"] == "skewed":
        p = torch.exp(3.0 * torch.randn(case["experts"], generator=g))
    to = torch.multinomial(p, case["rows"], replacement=True, generator=g)
    counts = torch.bincount(to, minlength=case["experts"])
    return [0] + torch.cumsum(counts, 0).tolist()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind.startswith("ln"):
        R, C, dt = case["rows"], case["cols"], TORCH[case["dtype"]]
        # the residual stream: a level and a size of its own in each column, a few columns much larger
        level, size = 0.25 + _normal(g, (C,), 0.2), 1.0 + 20.0 * (torch.rand(C, generator=g, device="cuda") < 0.01)
        x = (_normal(g, (R, C)) * size + level).to(dt)
        st = {"x": x, "gamma": (1.0 + _normal(g, (C,), 0.1)).to(dt), "beta": _normal(g, (C,), 0.1).to(dt),
              "residual": _normal(g, (R, C), 0.3).to(dt) if case["residual"] else None}
        if kind == "ln_backward":
            w = x.float()
            st["mean"] = w.mean(1)
            st["rstd"] = 1.0 / torch.sqrt((w - st["mean"][:, None]).square().mean(1) + EPS)
            st["dy"] = _normal(g, (R, C), 1e-2).to(dt)
        return {"case": case, **st}
    if kind == "adamw":
        sizes = _sizes(case)
        at = [0]  # every tensor of the program lives in one allocation, at a multiple of 256 values
        for n in sizes:
            at.append(at[-1] + -(-n // BLOCK) * BLOCK)
        live = torch.zeros(at[-1], dtype=torch.bool, device="cuda")
        for a, n in zip(at, sizes):
            live[a:a + n] = True
        rows = (at[-1] // BLOCK, BLOCK)
        size = torch.exp(_normal(g, (rows[0], 1))) * live.view(rows)  # tensors and rows learn at different rates
        p = (_normal(g, rows, 0.02) * live.view(rows)).view(-1)
        grad = (_normal(g, rows, 1e-3) * size).view(-1).to(TORCH[case["grad"]])
        m, v = _normal(g, rows, 3e-4) * size, (_normal(g, rows, 1e-3) * size).square()
        st = {"p": p, "grad": grad, "m": m.view(-1), "v": v.view(-1), "step": 100}
        if case["state"] == "8":
            root = v.sqrt()
            ms, vs = (torch.where(t > 0, t / 448.0, 1.0) for t in (m.abs().amax(1), root.amax(1)))
            st["m"], st["v"] = (m / ms[:, None]).to(E4).view(-1), (root / vs[:, None]).to(E4).view(-1)
            st["m_scale"], st["v_scale"] = ms, vs
        if case["copy"] != "none":
            st["copy"] = p.to(TORCH[case["copy"]])
        cut = lambda t, unit=1: [t[a // unit:a // unit + -(-n // unit)] for a, n in zip(at, sizes)]
        st["cut"] = {k: cut(t, BLOCK if "scale" in k else 1) for k, t in st.items() if k != "step"}
        return {"case": case, **st}
    R, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
    bounds = _bounds(case, seed)
    w = _normal(g, (E, N, K), 0.02) * torch.exp(0.3 * _normal(g, (E, 1, 1)))
    parts = [_codes(w[e], E4) for e in range(E)]
    st = {"case": case, "bounds": bounds, "offsets": torch.tensor(bounds, dtype=torch.int32, device="cuda"),
          "sw": torch.cat([s for _, s in parts])}
    x = _normal(g, (R, K))
    if kind == "experts_fwd":
        st["wq"] = torch.stack([q for q, _ in parts])
        st["xq"], st["sx"] = _codes(x, E4)
        return st
    dy = _normal(g, (R, N), 1e-3)
    st["wtq"] = torch.stack([_codes(w[e].t().contiguous(), E4)[0] for e in range(E)])
    st["dyq"], st["sdy"] = _codes(dy, E5)
    st["dytq"], st["xtq"] = _codes(dy.t().contiguous(), E5)[0], _codes(x.t().contiguous(), E4)[0]
    st["sx"] = _codes(x, E4)[1]
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return RUN[state["case"]["kind"]](state)


def _ln_forward(st):
    if own:
        import deepfuse_amd as df
        return df.layernorm_forward(st["x"], st["gamma"], st["beta"], EPS, residual=st["residual"])
    x = st["x"]
    s = x if st["residual"] is None else (x.float() + st["residual"].float()).to(x.dtype)
    w = s.float()
    mean = w.mean(1)
    c = w - mean[:, None]
    rstd = 1.0 / torch.sqrt(c.square().mean(1) + EPS)
    y = (c * rstd[:, None]) * st["gamma"].float() + st["beta"].float()
    return y.to(x.dtype), s, mean, rstd


def _ln_backward(st):
    if own:
        import deepfuse_amd as df
        return df.layernorm_backward(st["dy"], st["x"], st["gamma"], st["mean"], st["rstd"],
                                     dresidual=st["residual"])
    dy, rstd = st["dy"].float(), st["rstd"][:, None]
    xh = (st["x"].float() - st["mean"][:, None]) * rstd
    g = dy * st["gamma"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if st["residual"] is not None:
        dx = dx + st["residual"].float()
    return dx.to(st["x"].dtype), (dy * xh).sum(0), dy.sum(0)


def _bias_corrections(step):
    """1 - beta^step, beta^step and the difference rounded to 32 bits."""
    f = lambda v: torch.tensor(v, dtype=torch.float64).float()
    return [float(1.0 - f(float(f(b)) ** step)) for b in (BETA1, BETA2)]


def _adamw(st):
    st["step"] += 1
    eight, cut = st["case"]["state"] == "8", st["cut"]
    if own:
        import deepfuse_amd as df
        df.adamw_update(cut["p"], cut["grad"], cut["m"], cut["v"], st["step"], LR, BETA1, BETA2, ADAM_EPS, DECAY,
                        m_scales=cut.get("m_scale"), v_scales=cut.get("v_scale"), copies=cut.get("copy"))
        return {k: t for k, t in st.items() if k in ("p", "m", "v", "m_scale", "v_scale", "copy")}
    f = lambda v: torch.full((1,), v, dtype=torch.float32, device="cuda")  # constants in 32 bits, as the formula has them
    lr, b1, b2, one = f(LR), f(BETA1), f(BETA2), f(1.0)
    bc1, bc2 = (f(v) for v in _bias_corrections(st["step"]))
    g, m, v = st["grad"].float(), st["m"], st["v"]
    if eight:
        m = (m.float().view(-1, BLOCK) * st["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * st["v_scale"][:, None]).square().view(-1)
    m = b1 * m + (one - b1) * g
    v = b2 * v + (one - b2) * g * g
    st["p"].copy_(st["p"] * (one - lr * f(DECAY)) - lr * (m / bc1) / ((v / bc2).sqrt() + f(ADAM_EPS)))
    if "copy" in st:
        st["copy"].copy_(st["p"])
    if not eight:
        st["m"].copy_(m)
        st["v"].copy_(v)
        return {k: t for k, t in st.items() if k in ("p", "m", "v", "copy")}
    top, tiny, least = f(448.0), f(2.0 ** -126), f(2.0 ** -9)
    for name, x in (("m", m), ("v", v.sqrt())):
        x = x.view(-1, BLOCK)
        big = x.abs().amax(1)
        s = torch.where(big > 0, torch.maximum(big / top, tiny), one)
        q = (x / s[:, None]).clamp(-448.0, 448.0)
        if name == "v":
            q = torch.where((q > 0) & (q < least), least, q)
        st[name].copy_(q.view(-1).to(E4))
        st[name + "_scale"].copy_(s)
    return {k: t for k, t in st.items() if k in ("p", "m", "v", "m_scale", "v_scale", "copy")}


def _experts_fwd(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        return df.experts_fwd(st["xq"], st["wq"], st["offsets"], c["k"], st["sx"], st["sw"],
                              out_dtype=TORCH[c["dtype"]])
    x, w, b = st["xq"].view(E4).float()[:, :c["k"]], st["wq"].view(E4).float()[:, :, :c["k"]], st["bounds"]
    y = [(x[lo:hi] @ w[e].t()) * (st["sx"] * st["sw"][e]) for e, (lo, hi) in enumerate(zip(b, b[1:]))]
    return torch.cat(y).to(TORCH[c["dtype"]])


def _experts_bwd(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        return (df.experts_dx(st["dyq"], st["wtq"], st["offsets"], c["n"], st["sdy"], st["sw"],
                              out_dtype=TORCH[c["dtype"]]),
                df.experts_dw(st["dytq"], st["xtq"], st["offsets"], c["rows"], st["sdy"], st["sx"]))
    K, N, R, b = c["k"], c["n"], c["rows"], st["bounds"]
    dy, wt = st["dyq"].view(E5).float()[:, :N], st["wtq"].view(E4).float()[:, :, :N]
    dyt, xt = st["dytq"].view(E5).float()[:, :R], st["xtq"].view(E4).float()[:, :R]
    span = list(enumerate(zip(b, b[1:])))
    dx = torch.cat([(dy[lo:hi] @ wt[e].t()) * (st["sdy"] * st["sw"][e]) for e, (lo, hi) in span])
    dw = torch.stack([(dyt[:, lo:hi] @ xt[:, lo:hi].t()) * (st["sdy"] * st["sx"]) for e, (lo, hi) in span])
    return dx.to(TORCH[c["dtype"]]), dw


RUN = {"ln_forward": _ln_forward, "ln_backward": _ln_backward, "adamw": _adamw, "experts_fwd": _experts_fwd,
       "experts_bwd": _experts_bwd}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind.startswith("ln"):
        R, C, e = case["rows"], case["cols"], SIZE[case["dtype"]]
        if kind == "ln_forward":  # x (and residual) in, y (and the sum) out, gamma, beta, two statistics a row
            return {"bytes": R * C * e * (4 if case["residual"] else 2) + 2 * C * e + 8 * R, "flops": 8 * R * C}
        return {"bytes": R * C * e * (4 if case["residual"] else 3) + C * (e + 8) + 8 * R, "flops": 14 * R * C}
    if kind == "adamw":
        n = sum(_sizes(case))
        state = 24 if case["state"] == "32" else 8 + 4 + 16 / BLOCK  # p, m and v (and scales) read and written
        return {"bytes": int(n * (state + SIZE[case["grad"]] + (2 if case["copy"] != "none" else 0))), "flops": 18 * n}
    R, E, K, N, e = case["rows"], case["experts"], case["k"], case["n"], SIZE[case["dtype"]]
    used = min(E, R)  # experts without a row need no weights
    if kind == "experts_fwd":
        return {"bytes": R * K + used * N * K + R * N * e, "flops": 2 * R * N * K}
    return {"bytes": R * N + used * N * K + R * K * e + R * (N + K) + 4 * E * N * K, "flops": 4 * R * N * K}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _e4m3(x):
    """Nearest e4m3 value, ties to even, in 64 bits: steps of 2^(exponent - 3), of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    d = lambda k: st[k].double()
    if kind == "ln_forward":
        s = st["x"] if st["residual"] is None else (d("x") + d("residual")).to(st["x"].dtype)
        var, mean = torch.var_mean(s.double(), 1, correction=0)
        rstd = (var + EPS) ** -0.5
        return (s.double() - mean[:, None]) * rstd[:, None] * d("gamma") + d("beta"), s.double(), mean, rstd
    if kind == "ln_backward":
        # the gradient of sum(dy * y) through y = xh * gamma + beta, as the projection of g off 1 and xh
        xh, g = (d("x") - d("mean")[:, None]) * d("rstd")[:, None], d("dy") * d("gamma")
        n = case["cols"]
        dx = (g - (g.sum(1, keepdim=True) + xh * (g * xh).sum(1, keepdim=True)) / n) * d("rstd")[:, None]
        dx = dx if st["residual"] is None else dx + d("residual")
        return dx, (d("dy") * xh).sum(0), d("dy").sum(0)
    if kind == "adamw":
        t, eight = st["step"] + 1, case["state"] == "8"
        b1, b2, lr, eps, wd = (float(torch.tensor(v, dtype=torch.float32)) for v in (BETA1, BETA2, LR, ADAM_EPS, DECAY))
        m, v = d("m"), d("v")
        if eight:
            wide = lambda k: d(k + "_scale").repeat_interleave(BLOCK)
            m, v = m * wide("m"), (v * wide("v")) ** 2
        m.lerp_(d("grad"), 1 - b1)
        v.lerp_(d("grad") ** 2, 1 - b2)
        p = d("p") * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + eps)
        out = {"p": p, "m": m, "v": v}
        if eight:
            for k, x in (("m", m), ("v", v ** 0.5)):
                top = x.abs().view(-1, BLOCK).amax(1)
                s = torch.where(top > 0, top / 448, 1.0)
                q = x / s.repeat_interleave(BLOCK)
                out[k], out[k + "_scale"] = _e4m3(q if k == "m" else torch.where(q > 0, q.clamp(min=2.0 ** -9), q)), s
        if case["copy"] != "none":
            out["copy"] = p
        return out
    K, N, R = case["k"], case["n"], case["rows"]
    who = torch.repeat_interleave(torch.arange(case["experts"], device="cuda"), st["offsets"].diff().long())
    if kind == "experts_fwd":
        y = torch.empty(R, N, dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            w = st["wq"][e].view(E4).double()[:, :K] * d("sw")[e]
            y[who == e] = (st["xq"][who == e].view(E4).double()[:, :K] * d("sx")) @ w.T
        return y
    dx = torch.empty(R, K, dtype=torch.float64, device="cuda")
    dw = torch.empty(case["experts"], N, K, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        wt = st["wtq"][e].view(E4).double()[:, :N] * d("sw")[e]
        dx[who == e] = (st["dyq"][who == e].view(E5).double()[:, :N] * d("sdy")) @ wt.T
        mine = (who == e).double()
        dw[e] = (st["dytq"].view(E5).double()[:, :R] * mine * d("sdy")) @ (st["xtq"].view(E4).double()[:, :R].T * d("sx"))
    return dx, dw
