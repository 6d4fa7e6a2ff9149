"""fp8 with a scale per 128 values: what a block of a transformer built on deepfuse_amd does with it, in plain form too.

A case is a dict of plain values; its "kind" says which operator it runs:

  quantize      a matrix to fp8 codes with a scale per 128 values: of a row and, for the transposed codes, of a column,
                or (weights) per 128 x 128 square
  mm_fwd        a Linear's product on such codes, with its bias
  mm_bwd        the same Linear's dX and dW
  rms_forward   root-mean-square norm over rows, with the residual add in front of it; the output in the element type,
                or as codes with a scale per 128 columns
  rms_backward  its backward: dx (plus the residual path's gradient) and dgamma
  moe           a mixture-of-experts layer for a few tokens: the experts chosen from the router's logits, both Linears
                of each on e4m3 weights, the activation between them, the weighted sum

Scales are powers of two ("e8m0", one byte) or fp32 numbers ("f32").  Where `own` is false, run() computes in elementary
torch operations, in 32 bits; where it is true, it calls the library.  The sizes are those of GPT-2 small and GPT-2 XL
blocks, as bench.py and the tests run them, and odd ones.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
TOP = {"e4m3": 9, "e5m2": 16}  # fmax = 0.875 * 2^TOP
E8 = torch.float8_e8m0fnu
BLOCK = 128  # values that share a scale
EPS = 1e-5  # of the norm


def quantize(name, rows, cols, dtype="bf16", fmt="e4m3", square=False, both=True, scales="e8m0"):
    return {"name": name, "kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype, "fmt": fmt,
            "square": square, "both": both, "scales": scales}


def mm(name, kind, rows, k, n, dtype="bf16", grad="bf16", fmt="e4m3", bias=True, scales="e8m0"):
    return {"name": name, "kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "grad": grad, "fmt": fmt,
            "bias": bias, "scales": scales}


def rms(name, kind, rows, cols, dtype="bf16", residual=True, codes=True, scales="e8m0"):
    return {"name": name, "kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "residual": residual,
            "codes": codes, "scales": scales}


def moe(name, rows, experts, top, k, n, act="swiglu", dtype="bf16", scales="e8m0"):
    return {"name": name, "kind": "moe", "rows": rows, "experts": experts, "top": top, "k": k, "n": n, "act": act,
            "dtype": dtype, "scales": scales}


def listed():
    return [
        # a large model's activation on its way into fc2, for the forward and for dW
        quantize("quantize_xl", 16384, 6400),
        # an fp32 weight whose sizes are no multiples of anything, in squares, once a step
        quantize("quantize_weight_ragged", 1037, 771, dtype="f32", square=True),
        # a few sequences generating: qkv, bound by reading its weights
        mm("mm_fwd_decode", "mm_fwd", 16, 1600, 4800),
        # a large model's fc1 over a full batch
        mm("mm_fwd_xl", "mm_fwd", 16384, 1600, 6400),
        # its backward, 16-bit gradients
        mm("mm_bwd_xl", "mm_bwd", 16384, 1600, 6400),
        # a checkpoint's fp32 scales over a prompt of odd length, odd sizes, half precision
        mm("mm_fwd_ragged", "mm_fwd", 1000, 771, 1037, dtype="f16", scales="f32"),
        # one token of a small model being generated: all latency
        rms("rms_forward_token", "rms_forward", 1, 768),
        # a large model's norm over a full batch, in front of an fp8 Linear
        rms("rms_forward_xl", "rms_forward", 16384, 1600),
        # its backward
        rms("rms_backward_xl", "rms_backward", 16384, 1600),
        # a width that is no multiple of anything, in half precision, no residual path
        rms("rms_backward_ragged", "rms_backward", 1000, 771, dtype="f16", residual=False),
        # one token through two of 32 experts
        moe("moe_token", 1, 32, 2, 1600, 1600),
        # a batch of sequences generating, most experts taken by a few tokens each
        moe("moe_batch", 48, 32, 2, 1600, 1600),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: any number, or, as most models have them, a multiple of 64."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.4 else min(hi, max(64, (w + 32) // 64 * 64))


MOST = {"bytes": 4.2e8, "flops": 6.7e11}  # a drawn case stays below the largest listed ones


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if all(w[k] <= MOST[k] for k in MOST):
            return c


def _draw(rng):
    kind = rng.choice(["quantize", "mm_fwd", "mm_fwd", "mm_bwd", "rms_forward", "rms_backward", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    scales = rng.choice(["e8m0", "e8m0", "f32"])
    if kind == "quantize":
        c = quantize("", _log(rng, 1, 16384), _width(rng, 32, 6400), dtype, rng.choice(["e4m3", "e4m3", "e5m2"]),
                     rng.random() < 0.4, rng.random() < 0.6, scales)
    elif kind.startswith("mm"):
        c = mm("", kind, _log(rng, 1, 16384), _width(rng, 64, 6400), _width(rng, 64, 6400), dtype,
               rng.choice(["bf16", "f32"]), rng.choice(["e4m3", "e5m2"]), rng.random() < 0.5, scales)
    elif kind.startswith("rms"):
        c = rms("", kind, _log(rng, 1, 16384), _width(rng, 32, 6400), dtype, rng.random() < 0.6, rng.random() < 0.6,
                scales)
    else:
        experts = _log(rng, 2, 64)
        c = moe("", _log(rng, 1, 64), experts, min(experts, _log(rng, 1, 8)), _width(rng, 64, 2560),
                _width(rng, 64, 2560), rng.choice(["swiglu", "swiglu", "geglu", "gelu"]), rng.choice(["bf16", "f16"]),
                scales)
    del c["name"]
    return c


# ---- sizes, inputs ---------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _blocks(n):
    return -(-n // BLOCK)


def _stream(g, rows, cols):
    """The residual stream and what is made of it: a level and a size of its own in each column, a few much larger."""
    level = 0.25 + _normal(g, (cols,), 0.2)
    size = 1.0 + 20.0 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
    return _normal(g, (rows, cols)) * size + level


def _scales(most, fmt, kind):
    """A scale for each absmax: the smallest power of two that keeps it in range, or absmax / fmax."""
    if kind == "f32":
        return torch.where(most > 0, most / torch.full_like(most, FMAX[fmt]), 1.0)
    part, power = torch.frexp(most)
    e = power - TOP[fmt] + (part > 0.875)
    return (torch.where(most > 0, e, 0).clamp(-127, 127) + 127).to(torch.uint8).view(E8)


def _codes(x, fmt, kind, square=False):
    """fp8 codes of x, rows padded with zero codes to a multiple of 16, and the scales [blocks of columns, rows]."""
    rows, cols = x.shape
    w = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    most = w.abs().amax(2)
    if square:
        most = torch.nn.functional.pad(most, (0, 0, 0, -rows % BLOCK)).view(_blocks(rows), BLOCK, -1).amax(1)
        most = most.repeat_interleave(BLOCK, 0)[:rows]
    s = _scales(most, fmt, kind)
    q = (w / s.float()[:, :, None]).clamp(-FMAX[fmt], FMAX[fmt]).to(FP8[fmt]).view(rows, -1)
    return q[:, :cols + -cols % 16].contiguous(), _rowwise(s)


def _rowwise(s):
    """Scales [rows, blocks] as the products read them: [blocks, rows], each block's at a multiple of 16 bytes."""
    t = s.view(torch.uint8) if s.dtype == E8 else s
    out = torch.zeros(t.shape[1], t.shape[0] + -t.shape[0] % 16, dtype=t.dtype, device=t.device)
    out[:, :t.shape[0]] = t.t()
    return (out.view(E8) if s.dtype == E8 else out)[:, :t.shape[0]]


def _values(q, s, cols, wide=torch.float32):
    """What codes and scales stand for."""
    return q[:, :cols].to(wide) * s.to(wide).t().repeat_interleave(BLOCK, 1)[:, :cols]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    st = {"case": case}
    if kind == "quantize":
        x = _normal(g, (case["rows"], case["cols"]), 0.02) if case["square"] else _stream(g, case["rows"], case["cols"])
        st["x"] = x.to(TORCH[case["dtype"]])
        return st
    if kind.startswith("rms"):
        R, C, dt = case["rows"], case["cols"], TORCH[case["dtype"]]
        st["x"] = _stream(g, R, C).to(dt)
        st["gamma"] = (1.0 + _normal(g, (C,), 0.1)).to(dt)
        st["residual"] = _normal(g, (R, C), 0.3).to(dt) if case["residual"] else None
        if kind == "rms_backward":
            st["rstd"] = 1.0 / torch.sqrt(st["x"].float().square().mean(1) + EPS)
            st["dy"] = _normal(g, (R, C), 1e-2).to(dt)
        return st
    if kind == "moe":
        T, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
        up = N if case["act"] == "gelu" else 2 * N
        st["x"] = _normal(g, (T, K)).to(TORCH[case["dtype"]])
        st["logits"] = _normal(g, (T, E)) + _normal(g, (E,), 0.5)  # some experts are preferred
        for name, rows, cols in (("1", up, K), ("2", K, N)):
            made = [_codes(_normal(g, (rows, cols), 0.02), "e4m3", case["scales"], True) for _ in range(E)]
            st["w" + name] = torch.stack([q for q, _ in made])
            both = torch.stack([s.contiguous().view(torch.uint8) if s.dtype == E8 else s for _, s in made])
            pad = torch.nn.functional.pad(both, (0, -rows % 16)).contiguous()
            st["s" + name] = (pad.view(E8) if case["scales"] == "e8m0" else pad)[:, :, :rows]
        return st
    R, K, N, kinds = case["rows"], case["k"], case["n"], case["scales"]
    x, w = _stream(g, R, K), _normal(g, (N, K), 0.02)
    if kind == "mm_fwd":
        st["xq"], st["sx"] = _codes(x, "e4m3", kinds)
        st["wq"], st["sw"] = _codes(w, "e4m3", kinds, True)
        st["bias"] = _normal(g, (N,), 0.1).to(TORCH[case["dtype"]]) if case["bias"] else None
        return st
    dy = _normal(g, (R, N), 1e-3) * torch.exp(_normal(g, (R, 1)))  # tokens matter to different degrees
    st["wtq"], st["swt"] = _codes(w.t().contiguous(), "e4m3", kinds, True)
    st["dyq"], st["sdy"] = _codes(dy, case["fmt"], kinds)
    st["dytq"], st["sdyt"] = _codes(dy.t().contiguous(), case["fmt"], kinds)
    st["xtq"], st["sxt"] = _codes(x.t().contiguous(), "e4m3", kinds)
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return RUN[state["case"]["kind"]](state)


def _scale_dtype(case):
    return E8 if case["scales"] == "e8m0" else torch.float32


def _quantize(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        fmt = df.Fmt.E4M3 if c["fmt"] == "e4m3" else df.Fmt.E5M2
        q, s, qt, st_ = df.quantize_blocks(st["x"], fmt, want_qt=c["both"], square=c["square"],
                                           scale_dtype=_scale_dtype(c))
        out = {"q": q.view(FP8[c["fmt"]]), "s": s}
        return {**out, "qt": qt.view(FP8[c["fmt"]]), "st": st_} if c["both"] else out
    out = dict(zip(("q", "s"), _codes(st["x"], c["fmt"], c["scales"], c["square"])))
    if c["both"]:
        out.update(zip(("qt", "st"), _codes(st["x"].t(), c["fmt"], c["scales"], c["square"])))
    return out


def _mm_fwd(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        return df.gemm_blocks(st["xq"], st["sx"], st["wq"], st["sw"], c["k"], bias=st["bias"],
                              out_dtype=TORCH[c["dtype"]])
    y = _values(st["xq"], st["sx"], c["k"]) @ _values(st["wq"], st["sw"], c["k"]).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(TORCH[c["dtype"]])


def _mm_bwd(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        return (df.gemm_blocks(st["dyq"], st["sdy"], st["wtq"], st["swt"], c["n"], out_dtype=TORCH[c["dtype"]]),
                df.gemm_blocks(st["dytq"], st["sdyt"], st["xtq"], st["sxt"], c["rows"], out_dtype=TORCH[c["grad"]]))
    dx = _values(st["dyq"], st["sdy"], c["n"]) @ _values(st["wtq"], st["swt"], c["n"]).t()
    dw = _values(st["dytq"], st["sdyt"], c["rows"]) @ _values(st["xtq"], st["sxt"], c["rows"]).t()
    return dx.to(TORCH[c["dtype"]]), dw.to(TORCH[c["grad"]])


def _rms_forward(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        if not c["codes"]:
            return df.rmsnorm_forward(st["x"], st["gamma"], EPS, residual=st["residual"])
        q, sq, s, rstd = df.rmsnorm_quantize(st["x"], st["gamma"], EPS, residual=st["residual"],
                                             scale_dtype=_scale_dtype(c))
        return q.view(FP8["e4m3"]), sq, s, rstd
    x = st["x"]
    s = x if st["residual"] is None else (x.float() + st["residual"].float()).to(x.dtype)
    w = s.float()
    rstd = 1.0 / torch.sqrt(w.square().mean(1) + EPS)
    y = (w * rstd[:, None]) * st["gamma"].float()
    return (*_codes(y, "e4m3", c["scales"]), s, rstd) if c["codes"] else (y.to(x.dtype), s, rstd)


def _rms_backward(st):
    if own:
        import deepfuse_amd as df
        return df.rmsnorm_backward(st["dy"], st["x"], st["gamma"], st["rstd"], dresidual=st["residual"])
    dy, rstd = st["dy"].float(), st["rstd"][:, None]
    xh = st["x"].float() * rstd
    g = dy * st["gamma"].float()
    dx = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    if st["residual"] is not None:
        dx = dx + st["residual"].float()
    return dx.to(st["x"].dtype), (dy * xh).sum(0)


def _gelu(v):
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _act(h, act):
    if act == "gelu":
        return _gelu(h)
    gate, up = h.chunk(2, -1)
    return (gate / (1.0 + torch.exp(-gate)) if act == "swiglu" else _gelu(gate)) * up


def _chosen(logits, top):
    """The top experts of each token, ties to the lower index, and their share of a softmax over them."""
    best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    w = torch.exp(best[:, :top] - best[:, :1])
    return ids[:, :top].to(torch.int32), w / w.sum(1, keepdim=True)


def _moe(st):
    c = st["case"]
    if own:
        import deepfuse_amd as df
        return df.moe_layer(st["x"], st["logits"], st["w1"], st["s1"], st["w2"], st["s2"], c["top"],
                            activation=c["act"])
    ids, weights = _chosen(st["logits"], c["top"])
    x = st["x"].float()
    y = torch.zeros_like(x)
    of = lambda n, e, cols: _values(st["w" + n][e], st["s" + n][e], cols)
    if ids.numel() < c["experts"]:  # few pairs: take each one's weights
        pick = lambda t, i: t.view(torch.uint8).index_select(0, i)[0].view(t.dtype) if t.dtype != torch.float32 \
            else t.index_select(0, i)[0]
        for t in range(c["rows"]):
            for j in range(c["top"]):
                i = ids[t, j:j + 1]
                h = x[t] @ _values(pick(st["w1"], i), pick(st["s1"], i), c["k"]).t()
                w2 = _values(pick(st["w2"], i), pick(st["s2"], i), c["n"])
                y[t] += weights[t, j] * (_act(h, c["act"]) @ w2.t())
        return y.to(st["x"].dtype), ids, weights
    for e in range(c["experts"]):
        share = (weights * (ids == e)).sum(1, keepdim=True)
        y += share * (_act(x @ of("1", e, c["k"]).t(), c["act"]) @ of("2", e, c["n"]).t())
    return y.to(st["x"].dtype), ids, weights


RUN = {"quantize": _quantize, "mm_fwd": _mm_fwd, "mm_bwd": _mm_bwd, "rms_forward": _rms_forward,
       "rms_backward": _rms_backward, "moe": _moe}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind, sb = case["kind"], (1 if case["scales"] == "e8m0" else 4) / BLOCK  # of the scales, per code
    if kind == "quantize":
        n, copies = case["rows"] * case["cols"], 2 if case["both"] else 1
        return {"bytes": int(n * (SIZE[case["dtype"]] + copies * (1 + sb))), "flops": 3 * copies * n}
    if kind.startswith("rms"):
        R, C, e = case["rows"], case["cols"], SIZE[case["dtype"]]
        if kind == "rms_forward":  # x (and residual) in, the sum and y or its codes out, gamma, a statistic a row
            out = 1 + sb if case["codes"] else e
            return {"bytes": int(R * C * (e * (3 if case["residual"] else 1) + out)) + C * e + 4 * R, "flops": 6 * R * C}
        return {"bytes": R * C * e * (4 if case["residual"] else 3) + C * (e + 4) + 4 * R, "flops": 10 * R * C}
    if kind == "moe":
        T, K, N = case["rows"], case["k"], case["n"]
        used, up = min(case["experts"], T * case["top"]), 1 if case["act"] == "gelu" else 2  # experts that some token takes
        return {"bytes": int(used * (up + 1) * N * K * (1 + sb)) + T * (4 * K + 4 * case["experts"] + 8 * case["top"]),
                "flops": 2 * T * case["top"] * (up + 1) * N * K}
    R, K, N, e = case["rows"], case["k"], case["n"], SIZE[case["dtype"]]
    if kind == "mm_fwd":
        return {"bytes": int((R * K + N * K) * (1 + sb)) + R * N * e, "flops": 2 * R * N * K}
    return {"bytes": int((2 * R * N + N * K + R * K) * (1 + sb)) + R * K * e + N * K * SIZE[case["grad"]],
            "flops": 4 * R * N * K}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _nearest(x, fmt):
    """Nearest fp8 value, ties to even, in 64 bits: steps of 2^(exponent - bits), one size below the least normal."""
    bits, least = (3, -6) if fmt == "e4m3" else (2, -14)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least))) - bits)
    return (torch.round(x / step) * step).clamp(-FMAX[fmt], FMAX[fmt])


def _exact_codes(x, case, fmt, square=False):
    rows, cols = x.shape
    q = torch.zeros(rows, cols + -cols % 16, dtype=torch.float64, device="cuda")
    s = torch.ones(_blocks(cols), rows, dtype=torch.float64, device="cuda")
    for b in range(_blocks(cols)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        top = part.abs().amax(1)
        if square:
            for r in range(0, rows, BLOCK):
                top[r:r + BLOCK] = top[r:r + BLOCK].max()
        s[b] = top / FMAX[fmt]
        if case["scales"] == "e8m0":
            s[b] = torch.exp2(torch.ceil(torch.log2(s[b])))
        s[b][top == 0] = 1.0
        q[:, b * BLOCK:b * BLOCK + part.shape[1]] = _nearest(part / s[b][:, None], fmt)
    return q, s


def _wide(st, name, scale, cols, e=None):
    """Codes times scales in 64 bits, a block of columns at a time."""
    q, s = (st[name], st[scale]) if e is None else (st[name][e], st[scale][e])
    out = q[:, :cols].double()
    for b in range(_blocks(cols)):
        out[:, b * BLOCK:(b + 1) * BLOCK] *= s[b].double()[:, None]
    return out


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        x = st["x"].double()
        q, s = _exact_codes(x, case, case["fmt"], case["square"])
        if not case["both"]:
            return {"q": q, "s": s}
        qt, s_t = _exact_codes(x.t(), case, case["fmt"], case["square"])
        return {"q": q, "s": s, "qt": qt, "st": s_t}
    if kind == "mm_fwd":
        y = _wide(st, "xq", "sx", case["k"]) @ _wide(st, "wq", "sw", case["k"]).T
        return y if st["bias"] is None else y + st["bias"].double()
    if kind == "mm_bwd":
        return (_wide(st, "dyq", "sdy", case["n"]) @ _wide(st, "wtq", "swt", case["n"]).T,
                _wide(st, "dytq", "sdyt", case["rows"]) @ _wide(st, "xtq", "sxt", case["rows"]).T)
    if kind == "rms_forward":
        s = st["x"] if st["residual"] is None else (st["x"].double() + st["residual"].double()).to(st["x"].dtype)
        rstd = ((s.double() ** 2).sum(1) / case["cols"] + EPS) ** -0.5
        y = s.double() * rstd[:, None] * st["gamma"].double()
        return (*_exact_codes(y, case, "e4m3"), s.double(), rstd) if case["codes"] else (y, s.double(), rstd)
    if kind == "rms_backward":
        # the gradient of sum(dy * y) through y = xh * gamma, as what of g is orthogonal to xh
        rstd = st["rstd"].double()[:, None]
        xh, g = st["x"].double() * rstd, st["dy"].double() * st["gamma"].double()
        dx = (g - xh * ((g * xh).sum(1, keepdim=True) / case["cols"])) * rstd
        dx = dx if st["residual"] is None else dx + st["residual"].double()
        return dx, (st["dy"].double() * xh).sum(0)
    logits, x, top = st["logits"].double(), st["x"].double(), case["top"]
    ids = torch.argsort(-logits, dim=1, stable=True)[:, :top]
    weights = torch.softmax(logits.gather(1, ids), 1)
    y = torch.zeros_like(x)
    for e in ids.unique().tolist():
        who, place = torch.where(ids == e)
        h = x[who] @ _wide(st, "w1", "s1", case["k"], e).T
        if case["act"] == "swiglu":
            h = torch.nn.functional.silu(h[:, :case["n"]]) * h[:, case["n"]:]
        elif case["act"] == "geglu":
            h = torch.nn.functional.gelu(h[:, :case["n"]], approximate="tanh") * h[:, case["n"]:]
        else:
            h = torch.nn.functional.gelu(h, approximate="tanh")
        y[who] += weights[who, place][:, None] * (h @ _wide(st, "w2", "s2", case["n"], e).T)
    return y, None, weights
