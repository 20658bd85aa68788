"""What is measured of the 8-bit linear, the rotary positions and the residual norms: the cases, their inputs,
their plain form in elementary torch operations, and their values in 64 bits.

Operators
  fp8_linear  y = x W^T, x quantized to e4m3 per row and 128 values, W in e4m3 with one scale per 128 x 128
  fp8_vjp     its vector-Jacobian product: dx through the same weight, dW from x and dy quantized along the rows
  rope        rotary positions of q and k (two layouts, part of the head, scaled frequencies)
  rope_vjp    its vector-Jacobian product
  norm        h' = h + alpha gate rms(y) w_post, x = rms(h') w_pre (also with x as e4m3 rows)
  norm_vjp    its vector-Jacobian product
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 128
AMAX_MIN = 2.0 ** -100
EPS = 1e-6
THETA = 1e6


# ------------------------------------------------------------------------------------ cases ---

def listed():
    return [
        # one token through the q | k | v projection of the 896-wide block (decode: latency)
        {"name": "fp8 1x896->1152", "op": "fp8_linear", "M": 1, "K": 896, "N": 1152, "dtype": "bf16"},
        # sixteen sequences' tokens through a wide projection (decode: the weight's bytes)
        {"name": "fp8 16x8192->8192", "op": "fp8_linear", "M": 16, "K": 8192, "N": 8192, "dtype": "bf16"},
        # one eval batch (8 x 2048) through the gate projection of the 896-wide block
        {"name": "fp8 16384x896->4864", "op": "fp8_linear", "M": 16384, "K": 896, "N": 4864, "dtype": "bf16"},
        # a ragged prefill through a wide projection (tensor cores)
        {"name": "fp8 8191x4096->8192", "op": "fp8_linear", "M": 8191, "K": 4096, "N": 8192, "dtype": "f16"},
        # the gradients of the up projection for a micro-batch of 2 x 2047 positions
        {"name": "fp8 vjp 4094x896->4864", "op": "fp8_vjp", "M": 4094, "K": 896, "N": 4864, "dtype": "bf16"},
        # one decoded token at a far position, 14 query and 2 key heads
        {"name": "rope 1x(14+2)x64", "op": "rope", "T": 1, "nq": 14, "nk": 2, "hd": 64, "rot": 64, "layout": "half",
         "scaling": "none", "far": 1000000, "packed": True, "dtype": "bf16"},
        # one eval batch's q and k, read where the q | k | v projection wrote them
        {"name": "rope 16384x(14+2)x64", "op": "rope", "T": 16384, "nq": 14, "nk": 2, "hd": 64, "rot": 64,
         "layout": "half", "scaling": "none", "far": 2048, "packed": True, "dtype": "bf16"},
        # the gradient of a ragged long-context batch: pairs, half of the head, scaled frequencies
        {"name": "rope vjp 8191x(32+8)x128", "op": "rope_vjp", "T": 8191, "nq": 32, "nk": 8, "hd": 128, "rot": 64,
         "layout": "interleaved", "scaling": "yarn", "far": 131072, "packed": False, "dtype": "f16"},
        # one decoded token between two blocks
        {"name": "norm 1x896", "op": "norm", "T": 1, "H": 896, "gates": 1, "fp8": False, "dtype": "bf16"},
        # one eval batch between two blocks, straight into the 8-bit projection's rows
        {"name": "norm 16384x896 e4m3", "op": "norm", "T": 16384, "H": 896, "gates": 0, "fp8": True, "dtype": "bf16"},
        # its gradient with a gate per channel
        {"name": "norm vjp 16384x896", "op": "norm_vjp", "T": 16384, "H": 896, "gates": 1, "fp8": False,
         "dtype": "bf16"},
        # the gradient of three sequences with a gate each, an odd width
        {"name": "norm vjp 6141x5121", "op": "norm_vjp", "T": 6141, "H": 5121, "gates": 3, "fp8": False,
         "dtype": "f16"},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["fp8_linear", "fp8_linear", "fp8_vjp", "rope", "rope_vjp", "norm", "norm_vjp"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("fp8"):
        most = 8191 * 4096 * 8192 // (4 if op == "fp8_vjp" else 1)
        while True:
            M, K, N = _log(rng, 1, 16384), _log(rng, 64, 8192), _log(rng, 64, 8192)
            if rng.random() < 0.7:  # widths of projections; the others are any number
                K, N = max(64, K // 16 * 16), max(64, N // 16 * 16)
            if M * K * N <= most:
                return {"op": op, "M": M, "K": K, "N": N, "dtype": dtype}
    if op.startswith("rope"):
        hd = rng.choice([64, 80, 96, 128, 256])
        nk = rng.choice([1, 2, 4, 8])
        return {"op": op, "T": _log(rng, 1, 16384), "nq": nk * rng.choice([1, 2, 4, 7]), "nk": nk, "hd": hd,
                "rot": rng.choice([hd, hd, hd // 2, hd // 4 // 2 * 2]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                "far": _log(rng, 16384, 4000000), "packed": rng.random() < 0.5, "dtype": dtype}
    gates = rng.choice([0, 1, 1, 2, 4])
    T = _log(rng, 1, 16384)
    return {"op": op, "T": T * max(1, gates) if T * max(1, gates) <= 16384 else T // 4 * 4 or 4,
            "H": _log(rng, 64, 8192), "gates": gates, "fp8": op == "norm" and rng.random() < 0.3, "dtype": dtype}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("fp8"):
        M, N, K = case["M"], case["N"], case["K"]
        scales = 4 * -(-N // BLOCK) * -(-K // BLOCK)
        if case["op"] == "fp8_linear":
            return {"bytes": es * M * (K + N) + N * K + scales, "flops": 2 * M * N * K}
        return {"bytes": es * M * (2 * K + N) + N * K + scales + 4 * N * K, "flops": 4 * M * N * K}
    if case["op"].startswith("rope"):
        T, heads = case["T"], case["nq"] + case["nk"]
        return {"bytes": 2 * es * T * heads * case["hd"] + 4 * T, "flops": 6 * T * heads * (case["rot"] // 2)}
    T, H, G = case["T"], case["H"], case["gates"]
    params = es * H * (2 + G)
    if case["op"] == "norm":
        out = es + (1 + 4 / BLOCK if case["fp8"] else es)
        return {"bytes": T * H * (2 * es + out) + 8 * T + params, "flops": 12 * T * H}
    return {"bytes": 6 * es * T * H + 8 * T + params + 4 * H * (2 + G), "flops": 30 * T * H}


# ----------------------------------------------------------------------------------- inputs ---

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, cols, dtype):
    """Hidden states: a few channels far larger than the others, rows of different size."""
    x = _normal(g, rows, cols)
    x *= 1 + 15 * (torch.rand(cols, device="cuda", generator=g) < 0.01)
    x *= torch.exp(0.5 * _normal(g, rows, 1))
    return x.to(dtype)


def _scaling(case):
    return {"none": None,
            "linear": {"type": "linear", "factor": 4.0},
            "ntk": {"type": "ntk", "factor": 4.0},
            "yarn": {"type": "yarn", "factor": 8.0, "original": 16384},
            "bands": {"type": "bands", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}[case["scaling"]]


def prepare(case, seed):
    g, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    s = {"case": case}
    if op.startswith("fp8"):
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _activations(g, M, K, dt)
        # the weight as a checkpoint holds it: e4m3 values and a scale per 128 x 128
        s["codes"], s["scales"] = _quantize_blocks(0.03 * _normal(g, N, K))
        if op == "fp8_vjp":
            s["dy"] = (1e-3 * _activations(g, M, N, torch.float32)).to(dt)
            s["codes_t"] = s["codes"].view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn)
        if own:  # the layer that a program keeps: it holds these tensors
            from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
            s["linear"] = Fp8Linear(s["codes"], s["scales"], codes_t=s.get("codes_t"))
    elif op.startswith("rope"):
        T, nq, nk, hd = case["T"], case["nq"], case["nk"], case["hd"]
        if case["packed"]:
            rows = _normal(g, T, (nq + 2 * nk) * hd).to(dt)
            s["q"] = rows[:, :nq * hd].view(T, nq, hd)
            s["k"] = rows[:, nq * hd:(nq + nk) * hd].view(T, nk, hd)
        else:
            s["q"], s["k"] = _normal(g, T, nq, hd).to(dt), _normal(g, T, nk, hd).to(dt)
        start = torch.randint(0, case["far"], (1,), device="cuda", generator=g)
        s["positions"] = ((start + torch.arange(T, device="cuda")) % case["far"]).to(torch.int32)
        inv, factor = _frequencies(case["rot"], _scaling(case))
        s["inv_freq"], s["factor"] = torch.as_tensor(inv, device="cuda"), factor
        if own:  # the plan that a program keeps
            from gsq_rco_mlx_b200.common.rotary import Rotary
            s["rotary"] = Rotary(hd, theta=THETA, rotary_dim=case["rot"], layout=case["layout"],
                                 scaling=_scaling(case))
    else:
        T, H, G = case["T"], case["H"], case["gates"]
        s["h"], s["y"] = _activations(g, T, H, dt), _activations(g, T, H, dt)
        s["w_post"] = (1 + 0.1 * _normal(g, H)).to(dt)
        s["w_pre"] = (1 + 0.1 * _normal(g, H)).to(dt)
        s["gate"] = (0.5 + 0.2 * _normal(g, G, H)).to(dt) if G else None
        s["scale"] = 0.7
        if op == "norm_vjp":
            s["dh"], s["dx"] = (0.1 * _normal(g, T, H)).to(dt), (0.1 * _normal(g, T, H)).to(dt)
            f = _norm_plain(s)  # the row statistics that the forward pass returned
            s["stats"] = torch.stack([f["r_post"], f["r_pre"]]).reshape(2, T).contiguous()
    return s


# ------------------------------------------------------------------------------ plain forms ---

def _pad(x, rows, cols):
    r, c = -x.shape[0] % rows, -x.shape[1] % cols
    return torch.nn.functional.pad(x, (0, c, 0, r)) if r or c else x


def _scale_of(amax):
    """(448 / amax, amax / 448), each one division of two tensors (with a number it is a product by a reciprocal)."""
    most = amax.new_full((), 448.0)
    return most / amax, amax / most


def _quantize_rows(x):
    """e4m3 values [R, C] and scales [R, ceil(C / 128)] of x [R, C]."""
    R, C = x.shape
    b = _pad(x.float(), 1, BLOCK).view(R, -1, BLOCK)
    amax = b.abs().amax(2, keepdim=True).clamp(min=AMAX_MIN)
    r, scale = _scale_of(amax)
    return (b * r).view(R, -1)[:, :C].to(torch.float8_e4m3fn), scale.view(R, -1)


def _quantize_blocks(w):
    N, K = w.shape
    b = _pad(w.float(), BLOCK, BLOCK)
    b = b.view(b.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    amax = b.abs().amax((1, 3), keepdim=True).clamp(min=AMAX_MIN)
    r, scale = _scale_of(amax)
    q = (b * r).view(b.shape[0] * BLOCK, -1)[:N, :K]
    return q.contiguous().to(torch.float8_e4m3fn), scale.view(amax.shape[0], -1).contiguous()


def _rows_value(x):
    q, s = _quantize_rows(x)
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _blocks_value(q, s):
    return q.float() * s.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _frequencies(rot, scaling):
    """Inverse frequencies (64 bits) of the rot / 2 pairs, and the factor on cos and sin."""
    j = np.arange(0, rot, 2, dtype=np.float64)
    inv = THETA ** (-j / rot)
    if scaling is None:
        return inv, 1.0
    kind, f = scaling["type"], scaling["factor"]
    if kind == "linear":
        return inv / f, 1.0
    if kind == "ntk":
        return (THETA * f ** (rot / max(1, rot - 2))) ** (-j / rot), 1.0
    if kind == "yarn":
        at = lambda turns: rot * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1
    turns = scaling["original"] * inv / (2 * math.pi)
    keep = np.clip((turns - scaling["low"]) / (scaling["high"] - scaling["low"]), 0, 1)
    return (1 - keep) * inv / f + keep * inv, 1.0


def _rotate(x, cos, sin, rot, layout):
    """x [T, heads, hd] by cos, sin [T, 1, rot / 2]."""
    x = x.to(cos.dtype)
    r = x[..., :rot]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([r, x[..., rot:]], -1)


def _rope_plain(s, sign):
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * (sign * s["factor"])).float()
    c = s["case"]
    return {n: _rotate(s[n], cos, sin, c["rot"], c["layout"]).to(s[n].dtype) for n in ("q", "k")}


def _gate_rows(s, f):
    """The gate of each row: [T, H], [1, H] or 1."""
    if s["gate"] is None:
        return 1.0
    g = s["gate"].to(f)
    return g if g.shape[0] == 1 else g.repeat_interleave(s["h"].shape[0] // g.shape[0], 0)


def _norm_plain(s):
    h, y = s["h"].float(), s["y"].float()
    r_post = (y.square().mean(1, keepdim=True) + EPS).rsqrt()
    h2 = h + s["scale"] * _gate_rows(s, torch.float32) * (y * r_post * s["w_post"].float())
    r_pre = (h2.square().mean(1, keepdim=True) + EPS).rsqrt()
    return {"h2": h2, "x": h2 * r_pre * s["w_pre"].float(), "r_post": r_post, "r_pre": r_pre}


def _norm_vjp(s, f):
    """The gradients in type f: dh, dy, dw_post, dw_pre, dgate."""
    h, y, dh2, dx = (s[n].to(f) for n in ("h", "y", "dh", "dx"))
    a, b, g, alpha = s["w_post"].to(f), s["w_pre"].to(f), _gate_rows(s, f), s["scale"]
    r1 = (y.square().mean(1, keepdim=True) + EPS).rsqrt()
    yn = y * r1
    n = yn * a
    h2 = h + alpha * g * n
    r2 = (h2.square().mean(1, keepdim=True) + EPS).rsqrt()
    hn = h2 * r2
    u = dx * b
    d = dh2 + r2 * (u - hn * (u * hn).mean(1, keepdim=True))
    dn = alpha * g * d
    v = dn * a
    out = {"dh": d, "dy": r1 * (v - yn * (v * yn).mean(1, keepdim=True)),
           "dw_post": (dn * yn).sum(0), "dw_pre": (dx * hn).sum(0)}
    if s["gate"] is not None:
        G = s["gate"].shape[0]
        out["dgate"] = (alpha * d * n).view(G, -1, h.shape[1]).sum(1)
    return out


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        return _run_own(s, op)
    if op == "fp8_linear":
        return (_rows_value(s["x"]) @ _blocks_value(s["codes"], s["scales"]).t()).to(s["x"].dtype)
    if op == "fp8_vjp":
        dx = _rows_value(s["dy"]) @ _blocks_value(s["codes"], s["scales"])
        dw = _rows_value(s["dy"].t()) @ _rows_value(s["x"].t()).t()
        return {"dx": dx.to(s["x"].dtype), "dw": dw}
    if op.startswith("rope"):
        return _rope_plain(s, -1.0 if op == "rope_vjp" else 1.0)
    dt = s["h"].dtype
    if op == "norm":
        f = _norm_plain(s)
        out = {"h": f["h2"].to(dt)}
        if s["case"]["fp8"]:
            out["codes"], out["scales"] = _quantize_rows(f["x"])
        else:
            out["x"] = f["x"].to(dt)
        out["stats"] = torch.stack([f["r_post"], f["r_pre"]]).view(2, -1)
        return out
    f = _norm_vjp(s, torch.float32)
    return {n: v.to(dt) if n in ("dh", "dy") else v for n, v in f.items()}


def _run_own(s, op):
    if op == "fp8_linear":
        return s["linear"](s["x"])
    if op == "fp8_vjp":
        dx, dw = s["linear"].vjp(s["x"], s["dy"])
        return {"dx": dx, "dw": dw}
    if op == "rope":
        q, k = s["rotary"](s["q"], s["k"], s["positions"])
        return {"q": q, "k": k}
    if op == "rope_vjp":
        q, k = s["rotary"].vjp(s["q"], s["k"], s["positions"])
        return {"q": q, "k": k}
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    if op == "norm":
        h, x, stats = residual_norm(s["h"], s["y"], s["w_post"], s["w_pre"], gate=s["gate"], scale=s["scale"],
                                    eps=EPS, fp8=s["case"]["fp8"])
        if s["case"]["fp8"]:
            return {"h": h, "codes": x.codes, "scales": x.scales, "stats": stats}
        return {"h": h, "x": x, "stats": stats}
    g = residual_norm_vjp(s["h"], s["y"], s["w_post"], s["w_pre"], s["stats"], s["dh"], s["dx"], gate=s["gate"],
                          scale=s["scale"])
    return {n: v for n, v in g.items() if v is not None}


# ------------------------------------------------------------------------------------ exact ---

def _e4m3(v):
    """v (64 bits) to the nearest e4m3 value, ties to even: 3 fraction bits, least exponent -6, largest 448."""
    e = torch.frexp(v)[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_rows(x):
    """What the e4m3 rows of x [R, C] stand for; scale and reciprocal are 32-bit numbers of the format."""
    x = x.double()
    C = x.shape[1]
    out = []
    for a in range(0, C, BLOCK):
        b = x[:, a:a + BLOCK]
        m = b.abs().max(1, keepdim=True)[0].clamp(min=AMAX_MIN)
        s, r = (m / 448.0).float().double(), (448.0 / m).float().double()
        out.append(_e4m3((b * r).float().double()) * s)
    return torch.cat(out, 1)


def _exact_weight(s):
    w = s["codes"].float().double()
    for i in range(s["scales"].shape[0]):
        for j in range(s["scales"].shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= s["scales"][i, j].double()
    return w


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "fp8_linear":
        return _exact_rows(s["x"]) @ _exact_weight(s).t()
    if op == "fp8_vjp":
        dx = _exact_rows(s["dy"]) @ _exact_weight(s)
        dyt, xt = _exact_rows(s["dy"].t().contiguous()), _exact_rows(s["x"].t().contiguous())
        return {"dx": dx, "dw": dyt @ xt.t()}
    if op.startswith("rope"):
        # each pair as a complex number times factor * exp(+-i t)
        t = s["positions"].double()[:, None] * s["inv_freq"][None, :]
        turn = torch.polar(torch.full_like(t, s["factor"]), -t if op == "rope_vjp" else t)[:, None, :]
        out, rot = {}, case["rot"]
        for n in ("q", "k"):
            x = s[n].double()
            if case["layout"] == "half":
                z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
                r = torch.cat([z.real, z.imag], -1)
            else:
                z = torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn
                r = torch.view_as_real(z).flatten(-2)
            out[n] = torch.cat([r, x[..., rot:]], -1)
        return out
    T, H = s["h"].shape
    h, y = s["h"].double(), s["y"].double()
    g = None if s["gate"] is None else s["gate"].double()
    a, b = s["w_post"].double(), s["w_pre"].double()
    leaves = [t.requires_grad_(op == "norm_vjp") for t in (h, y, a, b)] + ([] if g is None else [g.requires_grad_()])
    with torch.set_grad_enabled(op == "norm_vjp"):
        rp = 1 / torch.sqrt((y * y).sum(1) / H + EPS)
        n = y * rp[:, None] * a
        if g is not None:
            n = (n.view(g.shape[0], -1, H) * g[:, None, :]).view(T, H)
        h2 = h + s["scale"] * n
        rq = 1 / torch.sqrt((h2 * h2).sum(1) / H + EPS)
        x = h2 * rq[:, None] * b
        if op == "norm":
            out = {"h": h2, "stats": torch.stack([rp, rq])}
            if case["fp8"]:
                # the codes (values of the format) and the scales that the 64-bit x gives
                pad = torch.nn.functional.pad(x, (0, -H % BLOCK)).view(T, -1, BLOCK)
                m = pad.abs().amax(2).clamp(min=AMAX_MIN)
                out["scales"] = m / 448.0
                out["codes"] = _e4m3(pad * (448.0 / m)[..., None]).view(T, -1)[:, :H]
            else:
                out["x"] = x
            return out
        d = torch.autograd.grad([h2, x], leaves, [s["dh"].double(), s["dx"].double()])
    names = ["dh", "dy", "dw_post", "dw_pre"] + ([] if g is None else ["dgate"])
    return dict(zip(names, d))
