"""The measured cases of the 4-bit block operators: microscaled quantisation
and product (``scmp_vit_b200.mx``), gated residual + norm
(``scmp_vit_b200.vit.residual_norm``) and the qkv split with multi-axis
rotary positions (``scmp_vit_b200.attention.split_qkv_rotary``).

``run`` computes a case in its plain form (elementary torch operations in 32
bits), or with ``own`` set through the package's entry points; ``exact``
computes it in 64 bits from the definitions, written apart from both.
"""
import math

import torch

own = False

EPS = 1e-6
BASE = 10000.0
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases

def _quantize(name, fmt, dtype, rows, dim):
    return {"name": name, "op": "quantize", "fmt": fmt, "dtype": dtype, "rows": rows, "dim": dim}


def _linear(name, fmt, dtype, rows, dim, features, bias):
    return {"name": name, "op": "linear", "fmt": fmt, "dtype": dtype, "rows": rows, "dim": dim,
            "features": features, "bias": bias}


def _norm(name, dtype, batch, tokens, dim, kind, post, gate, train):
    return {"name": name, "op": "norm", "dtype": dtype, "batch": batch, "tokens": tokens,
            "dim": dim, "kind": kind, "post": post, "gate": gate, "train": train}


def _rotary(name, dtype, batch, frames, height, width, heads, kv_heads, dims, interleaved, train):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "frames": frames,
            "height": height, "width": width, "heads": heads, "kv_heads": kv_heads, "dims": dims,
            "interleaved": interleaved, "train": train}


def listed():
    return [
        # one image's tokens on their way into a 4-bit projection
        _quantize("quantize_image", "mxfp4", "bf16", 257, 1024),
        # the hidden activations of 64 images, fp32 glue, the finer format
        _quantize("quantize_hidden_64", "nvfp4", "fp32", 64 * 257, 4096),
        # one token through fc1: the smallest call, latency
        _linear("linear_token", "mxfp4", "bf16", 1, 1024, 4096, True),
        # one image's output projection
        _linear("linear_image", "nvfp4", "fp16", 257, 1024, 1024, True),
        # fc1 of 64 images in the fp32 glue of the benchmark's ViT
        _linear("linear_fc1_64_fp32", "mxfp4", "fp32", 64 * 257, 1024, 4096, True),
        # fc2 of 128 images: the largest product
        _linear("linear_fc2_128", "mxfp4", "bf16", 128 * 257, 4096, 1024, True),
        # one image's residual add and second norm
        _norm("norm_image", "bf16", 1, 257, 1024, "layer", False, False, False),
        # 64 images: residual add, second norm straight into fc1's 4-bit codes
        {"name": "norm_linear_64", "op": "norm_linear", "fmt": "mxfp4", "dtype": "bf16",
         "batch": 64, "tokens": 257, "dim": 1024, "features": 4096, "kind": "layer"},
        # a training step's residual + norm, both directions, fp32
        _norm("norm_train_64_fp32", "fp32", 64, 257, 1024, "layer", False, False, True),
        # an EVA-width block with a norm on both sides and a gate per image
        _norm("norm_train_gated", "bf16", 16, 1025, 1408, "rms", True, True, True),
        # one image's q, k, v with (height, width) positions
        _rotary("rotary_image", "bf16", 1, 1, 16, 16, 16, 16, "32,32", True, False),
        # eight short clips, (time, height, width) positions, shared k/v heads, both directions
        _rotary("rotary_video_train", "bf16", 8, 8, 16, 16, 16, 4, "16,24,24", False, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "norm", "norm", "norm_linear", "rotary",
                     "rotary"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    if op == "quantize":
        case = _quantize("", fmt, dtype, _log(rng, 1, 16000), _log(rng, 32, 4096))
    elif op == "linear":
        dim = _log(rng, 32, 4096)
        if rng.random() < 0.5:  # the multiples of 32 that models have
            dim = max(32, dim // 32 * 32)
        case = _linear("", fmt, dtype, _log(rng, 1, 16000), dim, _log(rng, 48, 4096),
                       rng.random() < 0.5)
    elif op in ("norm", "norm_linear"):
        dim = _log(rng, 64, 4096)
        if rng.random() < 0.7:
            dim = dim // 32 * 32
        tokens = _log(rng, 1, 1500)
        batch = max(1, min(_log(rng, 1, 64), (16 << 20) // (dim * tokens)))
        kind = rng.choice(["layer", "rms"])
        if op == "norm":
            case = _norm("", dtype, batch, tokens, dim, kind, rng.random() < 0.5,
                         rng.random() < 0.5, rng.random() < 0.6)
        else:
            # 16-bit outputs: a sum's last bit decides which code a value at a
            # border takes, and fp32 outputs would show that choice
            case = {"op": op, "fmt": fmt, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch,
                    "tokens": tokens, "dim": dim, "features": _log(rng, 48, 4096), "kind": kind}
    else:
        heads = rng.choice([1, 2, 4, 8, 12, 16])
        kv_heads = rng.choice([h for h in (1, 2, 4, 8, 12, 16) if heads % h == 0])
        dims = rng.choice(["32,32", "16,24,24", "64", "20,20", "24,12", "40,40", "44,42,42"])
        frames = rng.choice([1, 1, 2, 5, 8]) if dims.count(",") == 2 else 1
        case = _rotary("", dtype, max(1, _log(rng, 1, 32) // frames), frames, rng.randint(1, 24),
                       rng.randint(1, 24), heads, kv_heads, dims, rng.random() < 0.5,
                       rng.random() < 0.5)
    case.pop("name", None)
    return case


def _head_dim(dims):
    return -(-sum(dims) // 8) * 8  # 40 -> 40, 36 -> 40: the last four stay unrotated


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["dim"]
        packed = n * (0.5 + (1 / 32 if case["fmt"] == "mxfp4" else 1 / 16))
        return {"bytes": n * size + packed + n * size, "flops": 0}
    if op == "linear":
        m, k, n = case["rows"], case["dim"], case["features"]
        packed = n * k * (0.5 + (1 / 32 if case["fmt"] == "mxfp4" else 1 / 16))
        return {"bytes": m * k * size + packed + m * n * size, "flops": 2 * m * n * k}
    if op in ("norm", "norm_linear"):
        n = case["batch"] * case["tokens"] * case["dim"]
        if op == "norm_linear":
            m, k, f = case["batch"] * case["tokens"], case["dim"], case["features"]
            packed = f * k * (0.5 + (1 / 32 if case["fmt"] == "mxfp4" else 1 / 16))
            return {"bytes": 3 * n * size + packed + m * f * size, "flops": 2 * m * f * k}
        # x, y -> r, h; with gradients dr, dh -> dx, dy too
        return {"bytes": (8 if case["train"] else 4) * n * size,
                "flops": (40 if case["train"] else 12) * n}
    dims = [int(d) for d in case["dims"].split(",")]
    tokens = case["frames"] * case["height"] * case["width"] + 1
    width = (case["heads"] + 2 * case["kv_heads"]) * _head_dim(dims)
    n = case["batch"] * tokens * width
    return {"bytes": (4 if case["train"] else 2) * n * size,
            "flops": (6 if case["train"] else 3) * n}


# ---------------------------------------------------------------- the inputs

def _activations(g, rows, dim, dtype):
    """Unit activations with a few strong channels, as a ViT's residual stream has."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    channel = torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    channel[:: max(1, dim // 5)] *= 12.0
    return (x * channel).to(dtype)


def _raw(case, seed):
    """Every input of a case before a program lays out its weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def leaf(t):
        return t.to(dtype).requires_grad_(bool(case.get("train")))

    s = {}
    if op in ("quantize", "linear"):
        s["x"] = _activations(g, case["rows"], case["dim"], dtype)
    if op in ("norm", "norm_linear"):
        rows, c = case["batch"] * case["tokens"], case["dim"]
        shape = (case["batch"], case["tokens"], c)
        s["x"] = leaf(_activations(g, rows, c, torch.float32).reshape(shape))
        s["y"] = leaf(randn(*shape) * 0.7 + 0.1)
        s["weight"] = leaf(1 + 0.2 * randn(c))
        s["norm_bias"] = leaf(0.1 * randn(c)) if case["kind"] == "layer" else None
        s["gamma"] = leaf(0.5 + 0.3 * randn(c))
        if case.get("post"):
            s["post_weight"] = leaf(1 + 0.2 * randn(c))
            s["post_bias"] = leaf(0.1 * randn(c)) if case["kind"] == "layer" else None
        if case.get("gate"):
            s["gate"] = leaf(randn(case["batch"], c))
        if case.get("train"):
            s["grad_r"] = randn(*shape).to(dtype)
            s["grad_h"] = randn(*shape).to(dtype)
    if op in ("linear", "norm_linear"):
        s["w"] = (0.02 * randn(case["features"], case["dim"])).clamp_(-0.04, 0.04).to(dtype)
        s["bias"] = (0.1 * randn(case["features"])).to(dtype) if case.get("bias", True) else None
    if op == "rotary":
        dims = [int(d) for d in case["dims"].split(",")]
        grid = [case["frames"], case["height"], case["width"]][-len(dims):]
        d = _head_dim(dims)
        coords = torch.cartesian_prod(*[torch.arange(n, device="cuda") for n in grid])
        coords = coords.reshape(-1, len(dims)) if len(dims) > 1 else torch.arange(
            case["height"] * case["width"], device="cuda").reshape(-1, 1)
        # the class token carries no position
        pos = torch.cat([torch.full((1, len(dims)), -1, device="cuda"), coords])
        if case["frames"] > 1 and len(dims) < 3:
            raise ValueError("frames need three axes")
        s["dims"], s["pos"] = dims, pos.to(torch.int32)
        s["sizes"] = [int(pos[:, a].max()) + 1 for a in range(len(dims))]
        n, width = pos.shape[0], (case["heads"] + 2 * case["kv_heads"]) * d
        s["qkv"] = leaf(randn(case["batch"], n, width))
        if case["train"]:
            for name, h in (("q", "heads"), ("k", "kv_heads"), ("v", "kv_heads")):
                s["grad_" + name] = randn(case["batch"], case[h], n, d).to(dtype)
    return s


def prepare(case, seed):
    s = _raw(case, seed)
    s["case"] = case
    if "w" in s:  # the weight is laid out once, the package's way or as the values it stands for
        w = s.pop("w")
        exp = _tensor_exp(w) if case["fmt"] == "nvfp4" else 0
        if own:
            from scmp_vit_b200 import mx
            s["weight4"] = mx.mx_quantize(w, case["fmt"], scale_exp=exp)
        else:
            s["weight4"] = _plain_quantize(w, case["fmt"], exp)
    if case["op"] == "rotary" and own:
        from scmp_vit_b200.attention import RotaryAxes
        s["axes"] = RotaryAxes(s["dims"], s["sizes"], base=BASE,
                               interleaved=case["interleaved"], device="cuda")
    return s


def _tensor_exp(w):
    """Power-of-two tensor scale that brings the largest block scale near e4m3's 448."""
    return int(math.floor(math.log2(float(w.abs().max()) / (6 * 448)))) + 1


# ---------------------------------------------------------------- the plain forms

def _plain_quantize(x, fmt, scale_exp=0):
    """The fp32 values that x's 4-bit codes stand for."""
    rows, k = x.shape
    block = 32 if fmt == "mxfp4" else 16
    pad = -k % block
    v = torch.nn.functional.pad(x.float(), (0, pad)).reshape(rows, -1, block)
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        exponent = torch.frexp(amax)[1] - 3  # floor(log2 amax) - 2
        exponent = torch.where(amax > 0, exponent.clamp(-127, 127), -127)
        step = torch.ldexp(torch.ones_like(amax), exponent)
    else:
        step = (amax * 2.0 ** -scale_exp / 6).clamp(max=448).to(torch.float8_e4m3fn).float()
        step = step * 2.0 ** scale_exp
    a = torch.where(step > 0, v.abs() / step, 0).clamp(max=6.0)
    # e2m1: steps of 1/2 below 2, of 1 below 4, of 2 up to 6; torch.round goes to even
    a = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a),
                                                              torch.round(a / 2) * 2))
    return (torch.copysign(a, v) * step).reshape(rows, -1)[:, :k]


def _plain_norm(v, kind):
    """(normalised v, 1 / deviation) in fp32."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * rstd, rstd


def _plain_norm_grad(dn, n, rstd, kind):
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - dn.mean(-1, keepdim=True)
    return d * rstd


def _plain_residual(s, kind, dtype):
    x, y = s["x"].float(), s["y"].float()
    z, m, rstd_y = y, None, None
    if s.get("post_weight") is not None:
        m, rstd_y = _plain_norm(y, kind)
        z = m * s["post_weight"].float()
        if s["post_bias"] is not None:
            z = z + s["post_bias"].float()
    scale = s["gamma"].float()
    gate = s["gate"].float().unsqueeze(1) if s.get("gate") is not None else None
    both = scale if gate is None else scale * gate
    r = (x + z * both).to(dtype)
    n, rstd = _plain_norm(r.float(), kind)
    h = n * s["weight"].float()
    if s["norm_bias"] is not None:
        h = h + s["norm_bias"].float()
    return r, h, (n, rstd, z, m, rstd_y, scale, gate, both)


def _plain_norm_case(s, case):
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    r, h, (n, rstd, z, m, rstd_y, scale, gate, both) = _plain_residual(s, kind, dtype)
    out = {"r": r, "h": h.to(dtype)}
    if not case["train"]:
        return out
    dh, c = s["grad_h"].float(), case["dim"]
    g = s["grad_r"].float() + _plain_norm_grad(dh * s["weight"].float(), n, rstd, kind)
    out["x"] = g
    out["weight"] = (dh * n).reshape(-1, c).sum(0)
    if s["norm_bias"] is not None:
        out["norm_bias"] = dh.reshape(-1, c).sum(0)
    gz = (g * z).sum(1)
    out["gamma"] = (gz if gate is None else gz * gate.squeeze(1)).sum(0)
    if gate is not None:
        out["gate"] = gz * scale
    dz = g * both
    if m is not None:
        out["post_weight"] = (dz * m).reshape(-1, c).sum(0)
        if s["post_bias"] is not None:
            out["post_bias"] = dz.reshape(-1, c).sum(0)
        dz = _plain_norm_grad(dz * s["post_weight"].float(), m, rstd_y, kind)
    out["y"] = dz
    return {k: v.to(dtype) for k, v in out.items()}


def _plain_rotary_tables(s):
    """cos and sin [tokens, rotated pairs] in fp32; the angles need 64 bits."""
    angles = []
    for a, d in enumerate(s["dims"]):
        freq = BASE ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angles.append(s["pos"][:, a:a + 1].clamp(min=0).double() * freq)
    angle = torch.cat(angles, -1)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _pair_index(dims, interleaved):
    first, second, base = [], [], 0
    for d in dims:
        at = torch.arange(d // 2, device="cuda")
        first.append(base + (2 * at if interleaved else at))
        second.append(base + (2 * at + 1 if interleaved else at + d // 2))
        base += d
    return torch.cat(first), torch.cat(second)


def _plain_rotate(t, cos, sin, first, second):
    """t [B, H, N, D] in fp32, each pair turned by its token's angle."""
    u, v = t[..., first], t[..., second]
    out = t.clone()
    out[..., first] = u * cos - v * sin
    out[..., second] = v * cos + u * sin
    return out


def _plain_rotary(s, case):
    dtype = DTYPES[case["dtype"]]
    h, hk, d = case["heads"], case["kv_heads"], _head_dim(s["dims"])
    cos, sin = _plain_rotary_tables(s)
    first, second = _pair_index(s["dims"], case["interleaved"])
    b, n, _ = s["qkv"].shape
    heads = s["qkv"].float().reshape(b, n, h + 2 * hk, d).transpose(1, 2)
    q, k, v = heads.split([h, hk, hk], 1)
    out = {"q": _plain_rotate(q, cos, sin, first, second).to(dtype),
           "k": _plain_rotate(k, cos, sin, first, second).to(dtype),
           "v": v.to(dtype).contiguous()}
    if case["train"]:
        dq = _plain_rotate(s["grad_q"].float(), cos, -sin, first, second)
        dk = _plain_rotate(s["grad_k"].float(), cos, -sin, first, second)
        grad = torch.cat([dq, dk, s["grad_v"].float()], 1).transpose(1, 2)
        out["qkv"] = grad.reshape(b, n, -1).to(dtype)
    return out


@torch.no_grad()
def _plain(s):
    case = s["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "quantize":
        return _plain_quantize(s["x"], case["fmt"]).to(dtype)
    if op == "linear":
        y = _plain_quantize(s["x"], case["fmt"]) @ s["weight4"].t()
        return (y if s["bias"] is None else y + s["bias"].float()).to(dtype)
    if op == "norm":
        return _plain_norm_case(s, case)
    if op == "norm_linear":
        r, h, _ = _plain_residual(s, case["kind"], dtype)
        y = _plain_quantize(h.reshape(-1, case["dim"]), case["fmt"]) @ s["weight4"].t()
        y = (y + s["bias"].float()).to(dtype)
        return {"r": r, "out": y.reshape(case["batch"], case["tokens"], -1)}
    return _plain_rotary(s, case)


# ---------------------------------------------------------------- the package's calls

NORM_LEAVES = ("x", "y", "weight", "norm_bias", "gamma", "gate", "post_weight", "post_bias")


def _own(s):
    case = s["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "quantize":
        from scmp_vit_b200 import mx
        return mx.mx_quantize(s["x"], case["fmt"]).dequantize(dtype)
    if op == "linear":
        from scmp_vit_b200 import mx
        return mx.mx_matmul(s["x"], s["weight4"], bias=s["bias"])
    if op in ("norm", "norm_linear"):
        from scmp_vit_b200 import vit
        r, h = vit.residual_norm(
            s["x"], s["y"], s["weight"], s["norm_bias"], kind=case["kind"], eps=EPS,
            gamma=s["gamma"], gate=s.get("gate"), post_weight=s.get("post_weight"),
            post_bias=s.get("post_bias"), quantize=case.get("fmt"))
        if op == "norm_linear":
            from scmp_vit_b200 import mx
            return {"r": r, "out": mx.mx_matmul(h, s["weight4"], bias=s["bias"],
                                                out_dtype=dtype)}
        out = {"r": r, "h": h}
        if case["train"]:
            names = [n for n in NORM_LEAVES if s.get(n) is not None]
            grads = torch.autograd.grad((r, h), [s[n] for n in names],
                                        (s["grad_r"], s["grad_h"]))
            out.update(zip(names, grads))
        return out
    from scmp_vit_b200.attention import split_qkv_rotary
    q, k, v = split_qkv_rotary(s["qkv"], case["heads"], s["axes"], s["pos"],
                               num_kv_heads=case["kv_heads"], transpose_v=False)
    out = {"q": q, "k": k, "v": v}
    if case["train"]:
        (out["qkv"],) = torch.autograd.grad(
            (q, k, v), (s["qkv"],), (s["grad_q"], s["grad_k"], s["grad_v"]))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- 64 bits, from the definitions

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_codes(x, fmt, scale_exp=0):
    """The nearest representable values by a search over their borders; a
    value on a border takes the even code."""
    x = x.double()
    rows, k = x.shape
    block = 32 if fmt == "mxfp4" else 16
    nb = -(-k // block)
    padded = torch.zeros(rows, nb * block, dtype=torch.float64, device=x.device)
    padded[:, :k] = x
    v = padded.view(rows, nb, block)
    amax = v.abs().max(-1, keepdim=True).values
    if fmt == "mxfp4":
        e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140)))
        # log2 may round at a power of two: settle it by comparison
        e = torch.where(torch.exp2(e) > amax, e - 1, e)
        e = torch.where(torch.exp2(e + 1) <= amax, e + 1, e)
        step = torch.exp2((e - 2).clamp(min=-127))
    else:
        want = amax / 6 / 2.0 ** scale_exp
        grid = [i * 2.0 ** -9 for i in range(8)]
        grid += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
        grid = torch.tensor(grid[:127], dtype=torch.float64, device=x.device)  # up to 448
        step = grid[_nearest(want, grid)] * 2.0 ** scale_exp
    values = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    ratio = torch.where(step > 0, v.abs() / torch.where(step > 0, step, 1.0), 0.0)
    q = values[_nearest(ratio, values)] * step
    return torch.where(v < 0, -q, q).view(rows, -1)[:, :k]


def _nearest(v, grid):
    """Index of the nearest entry of a sorted grid, the even one between two."""
    border = (grid[1:] + grid[:-1]) / 2
    low = torch.searchsorted(border, v.contiguous(), right=False)  # borders below v
    high = torch.searchsorted(border, v.contiguous(), right=True)  # borders up to v
    return torch.where((low != high) & (low % 2 == 1), high, low)


def _exact_normed(v, kind):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    dev = torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + EPS)
    return (v - mean) / dev, dev


def _exact_back(grad, n, dev, kind):
    out = grad - n * (grad * n).mean(-1, keepdim=True)
    return (out - (grad.mean(-1, keepdim=True) if kind == "layer" else 0)) / dev


def _exact_norm(s, case):
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    t = {k: (v.detach().double() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
    one = torch.ones((), dtype=torch.float64, device="cuda")
    gate = t["gate"][:, None, :] if t.get("gate") is not None else one
    if t.get("post_weight") is not None:
        m, dev_y = _exact_normed(t["y"], kind)
        z = m * t["post_weight"] + (t["post_bias"] if t["post_bias"] is not None else 0)
    else:
        z = t["y"]
    r = (t["x"] + z * t["gamma"] * gate).to(dtype).double()
    n, dev = _exact_normed(r, kind)
    out = {"r": r, "h": n * t["weight"] + (t["norm_bias"] if t["norm_bias"] is not None else 0)}
    if not case.get("train"):
        return out
    dh = t["grad_h"]
    g = t["grad_r"] + _exact_back(dh * t["weight"], n, dev, kind)
    out["x"], out["weight"] = g, (dh * n).sum((0, 1))
    if t["norm_bias"] is not None:
        out["norm_bias"] = dh.sum((0, 1))
    out["gamma"] = (g * z * gate).sum((0, 1))
    if t.get("gate") is not None:
        out["gate"] = (g * z * t["gamma"]).sum(1)
    out["y"] = g * t["gamma"] * gate
    if t.get("post_weight") is not None:
        out["post_weight"] = (out["y"] * m).sum((0, 1))
        if t["post_bias"] is not None:
            out["post_bias"] = out["y"].sum((0, 1))
        out["y"] = _exact_back(out["y"] * t["post_weight"], m, dev_y, kind)
    return out


def _exact_rotary(s, case):
    """Each pair as a complex number, turned by e^(i angle)."""
    h, hk, d = case["heads"], case["kv_heads"], _head_dim(s["dims"])
    b, n, _ = s["qkv"].shape
    turn = torch.ones(n, d // 2, dtype=torch.complex128, device="cuda")
    order, base, at = [], 0, 0
    for a, da in enumerate(s["dims"]):
        for i in range(da // 2):
            angle = s["pos"][:, a].double() * math.pow(BASE, -2.0 * i / da)
            angle = torch.where(s["pos"][:, a] < 0, 0.0, angle)
            turn[:, at] = torch.polar(torch.ones_like(angle), angle)
            order += [base + 2 * i, base + 2 * i + 1] if case["interleaved"] else [
                base + i, base + i + da // 2]
            at, base = at + 1, base + (da if i == da // 2 - 1 else 0)
    order += list(range(base, d))
    order = torch.tensor(order, device="cuda")
    back = torch.argsort(order)

    def rotate(x, by):
        c = torch.view_as_complex(x.double()[..., order].reshape(*x.shape[:-1], d // 2, 2))
        return torch.view_as_real(c * by).reshape(x.shape)[..., back]

    x = s["qkv"].detach().reshape(b, n, h + 2 * hk, d).permute(0, 2, 1, 3)
    out = {"q": rotate(x[:, :h], turn), "k": rotate(x[:, h:h + hk], turn),
           "v": x[:, h + hk:].double()}
    if case["train"]:
        parts = [rotate(s["grad_q"], turn.conj()), rotate(s["grad_k"], turn.conj()),
                 s["grad_v"].double()]
        out["qkv"] = torch.cat(parts, 1).permute(0, 2, 1, 3).reshape(b, n, -1)
    return out


@torch.no_grad()
def exact(case, seed):
    s = _raw(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_codes(s["x"], case["fmt"])
    if op in ("linear", "norm_linear"):
        exp = _tensor_exp(s["w"]) if case["fmt"] == "nvfp4" else 0
        w = _exact_codes(s["w"], case["fmt"], exp)
        bias = s["bias"].double() if s["bias"] is not None else 0
        if op == "linear":
            return _exact_codes(s["x"], case["fmt"]) @ w.t() + bias
        t = _exact_norm(s, case)
        codes = _exact_codes(t["h"].reshape(-1, case["dim"]), case["fmt"])
        out = codes @ w.t() + bias
        return {"r": t["r"], "out": out.reshape(case["batch"], case["tokens"], -1)}
    if op == "norm":
        return _exact_norm(s, case)
    return _exact_rotary(s, case)
