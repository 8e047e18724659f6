"""The measured cases of the operators of a block trained and served in 8 bits:
the linear in 8-bit floating point with a scale per block of 128
(``scmp_vit_b200.fp8``), the qkv split with norms of queries and keys and
multi-axis rotary positions (``scmp_vit_b200.attention.split_qkv_norm``) and
dropout from a counter-based generator (``scmp_vit_b200.vit.dropout``).

``run`` computes a case in its plain form (elementary torch operations in 32
bits), or with ``own`` set through the package's entry points; ``exact``
computes it in 64 bits from the definitions, written apart from both.
"""
import math

import torch

own = False

EPS = 1e-6
BASE = 10000.0
BLOCK = 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases

def _linear(name, dtype, rows, dim, features, bias, train):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "dim": dim,
            "features": features, "bias": bias, "train": train}


def _qkv(name, dtype, batch, frames, height, width, cls, heads, kv_heads, head_dim, dims,
         interleaved, kind, train):
    return {"name": name, "op": "qkv", "dtype": dtype, "batch": batch, "frames": frames,
            "height": height, "width": width, "cls": cls, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dims": dims, "interleaved": interleaved, "kind": kind,
            "train": train}


def _dropout(name, dtype, batch, tokens, dim, p, per, residual, train):
    return {"name": name, "op": "dropout", "dtype": dtype, "batch": batch, "tokens": tokens,
            "dim": dim, "p": p, "per": per, "residual": residual, "train": train}


def listed():
    return [
        # one token through fc1: the smallest product, latency
        _linear("linear_token", "bf16", 1, 1024, 4096, True, False),
        # one image's output projection
        _linear("linear_image", "fp16", 257, 1024, 1024, True, False),
        # fc1 of 64 images
        _linear("linear_fc1_64", "bf16", 64 * 257, 1024, 4096, True, False),
        # a training step of a narrow projection with odd sizes, fp32 parameters
        _linear("linear_train_odd_fp32", "fp32", 4 * 197, 1000, 333, True, True),
        # a training step of fc2, 64 images: the largest product
        _linear("linear_train_fc2_64", "bf16", 64 * 257, 4096, 1024, True, True),
        # the next token of 32 sequences, shared k/v heads: the smallest split
        _qkv("qkv_token", "bf16", 32, 1, 1, 1, 0, 16, 4, 64, "64", False, "rms", False),
        # one image's q, k, v with (height, width) positions
        _qkv("qkv_image", "bf16", 1, 1, 16, 16, 1, 16, 16, 64, "32,32", True, "rms", False),
        # a training step of 64 images, layer norms with biases, fp32 glue
        _qkv("qkv_train_64_fp32", "fp32", 64, 1, 16, 16, 1, 16, 16, 64, "32,32", True, "layer",
             True),
        # a training step of eight short clips, (time, height, width), shared k/v heads
        _qkv("qkv_video_train", "bf16", 8, 8, 16, 16, 0, 16, 4, 64, "16,24,24", False, "rms",
             True),
        # one image's branch output on its way into the residual stream
        _dropout("dropout_image", "fp32", 1, 257, 1024, 0.1, "element", True, True),
        # a training step's hidden activations, 64 images
        _dropout("dropout_hidden_64", "bf16", 64, 257, 4096, 0.1, "element", False, True),
        # stochastic depth: 64 images, one draw each, with the residual add
        _dropout("drop_path_64", "fp32", 64, 257, 1024, 0.2, "sample", True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "qkv", "qkv", "dropout"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "linear":
        dim, features = _log(rng, 32, 4096), _log(rng, 32, 4096)
        if rng.random() < 0.5:  # the multiples of 32 that models have
            dim, features = max(32, dim // 32 * 32), max(32, features // 32 * 32)
        train = rng.random() < 0.5
        rows = _log(rng, 1, 16000)
        case = _linear("", dtype, min(rows, (64 * 257 << 22) // (dim * features)), dim, features,
                       rng.random() < 0.5, train)
    elif op == "qkv":
        heads = rng.choice([1, 2, 4, 8, 12, 16])
        kv_heads = rng.choice([h for h in (1, 2, 4, 8, 12, 16) if heads % h == 0])
        head_dim, dims = rng.choice([(64, "32,32"), (64, "16,24,24"), (64, "64"), (40, "20,20"),
                                     (48, "24,12"), (80, "40,40"), (128, "44,42,42"), (96, ""),
                                     (256, "128,128"), (36, "18")])
        frames = rng.choice([1, 1, 2, 5, 8]) if dims.count(",") == 2 else 1
        case = _qkv("", dtype, max(1, _log(rng, 1, 32) // frames), frames, rng.randint(1, 24),
                    rng.randint(1, 24), rng.randint(0, 1), heads, kv_heads, head_dim, dims,
                    rng.random() < 0.5, rng.choice(["rms", "layer"]), rng.random() < 0.5)
        tokens = case["batch"] * (case["frames"] * case["height"] * case["width"] + case["cls"])
        most = 64 * 257 * 48 * 64 // (tokens * (heads + 2 * kv_heads) * head_dim)
        if most < 1:
            case["batch"] = 1
    else:
        dim = _log(rng, 1, 4096)
        tokens = _log(rng, 1, 1500)
        batch = max(1, min(_log(rng, 1, 64), (64 * 257 * 1024) // (dim * tokens)))
        case = _dropout("", dtype, batch, tokens, dim, rng.choice([0.0, 0.05, 0.1, 0.5, 0.9]),
                        rng.choice(["element", "element", "row", "sample"]), rng.random() < 0.5,
                        rng.random() < 0.5)
    case.pop("name", None)
    return case


def _tokens(case):
    return case["frames"] * case["height"] * case["width"] + case["cls"]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "linear":
        m, k, n = case["rows"], case["dim"], case["features"]
        if case["train"]:  # x, W, b, dy -> y, dx, dW, db
            return {"bytes": 2 * size * (m * k + n * k + m * n + n * case["bias"]),
                    "flops": 6 * m * n * k}
        return {"bytes": m * k * size + n * k * (1 + 1 / BLOCK) + m * n * size,
                "flops": 2 * m * n * k}
    if op == "qkv":
        h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        tokens = case["batch"] * _tokens(case)
        qk, v = tokens * (h + hk) * d, tokens * hk * d
        return {"bytes": size * (2 * (qk + v) * (2 if case["train"] else 1)),
                "flops": (30 if case["train"] else 10) * qk}
    n = case["batch"] * case["tokens"] * case["dim"]
    passes = 2 + case["residual"] + 2 * case["train"]
    return {"bytes": passes * n * size, "flops": 2 * n * (2 if case["train"] else 1)}


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
        return t.to(dtype).requires_grad_(bool(case["train"]))

    s = {}
    if op == "linear":
        s["x"] = leaf(_activations(g, case["rows"], case["dim"], torch.float32))
        s["w"] = leaf((0.02 * randn(case["features"], case["dim"])).clamp_(-0.04, 0.04))
        s["b"] = leaf(0.1 * randn(case["features"])) if case["bias"] else None
        if case["train"]:  # gradients of very different sizes per token
            s["grad"] = (randn(case["rows"], case["features"])
                         * torch.exp(randn(case["rows"], 1)) * 1e-2).to(dtype)
    elif op == "qkv":
        dims = [int(d) for d in case["dims"].split(",")] if case["dims"] else []
        h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        b, n = case["batch"], _tokens(case)
        s["qkv"] = leaf(_activations(g, b * n, (h + 2 * hk) * d, torch.float32).reshape(b, n, -1))
        for name in ("q", "k"):
            s[name + "_weight"] = leaf(1 + 0.2 * randn(d))
            s[name + "_bias"] = leaf(0.1 * randn(d)) if case["kind"] == "layer" else None
        s["dims"] = dims
        if dims:
            grid = [case["frames"], case["height"], case["width"]][-len(dims):]
            if len(dims) == 1:
                grid = [case["height"] * case["width"]]
            at = torch.meshgrid(*[torch.arange(m, device="cuda") for m in grid], indexing="ij")
            at = torch.stack([a.reshape(-1) for a in at], -1)
            if case["frames"] * case["height"] * case["width"] == 1:
                # the next token of each sequence: every one at a place of its own
                at = torch.randint(0, 1024, (b, 1, len(dims)), generator=g, device="cuda")
                head = at.new_full((b, case["cls"], len(dims)), -1)
                pos = torch.cat([head, at], 1)
            else:  # the class token carries no position
                pos = torch.cat([at.new_full((case["cls"], len(dims)), -1), at])
            s["pos"] = pos.to(torch.int32)
            s["sizes"] = [1024 if pos.dim() == 3 else m for m in grid] if len(dims) > 1 else [
                max(1024, grid[0])]
        if case["train"]:
            for name, m in (("q", h), ("k", hk), ("v", hk)):
                s["grad_" + name] = randn(b, m, n, d).to(dtype)
    else:
        shape = (case["batch"], case["tokens"], case["dim"])
        s["x"] = leaf(randn(*shape))
        s["residual"] = leaf(4 * randn(*shape)) if case["residual"] else None
        s["seed"] = int(torch.randint(1, 1 << 62, (), generator=g, device="cuda"))
        s["offset"] = int(torch.randint(0, 1 << 40, (), generator=g, device="cuda"))
        if case["train"]:
            s["grad"] = randn(*shape).to(dtype)
    return s


def prepare(case, seed):
    s = _raw(case, seed)
    s["case"] = case
    if case["op"] == "linear" and not case["train"]:
        # the weight is laid out once, the package's way or as the values it stands for
        w = s.pop("w")
        if own:
            from scmp_vit_b200 import fp8
            s["weight8"] = fp8.fp8_quantize(w, "square")
        else:
            s["weight8"] = _plain_square(w)
    if case["op"] == "qkv" and s["dims"] and own:
        from scmp_vit_b200.attention import RotaryAxes
        s["axes"] = RotaryAxes(s["dims"], s["sizes"], base=BASE,
                               interleaved=case["interleaved"], device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_codes(v, amax):
    """The fp32 values that v's 8-bit codes stand for under power-of-two steps."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)  # 448 = 0.875 2^9
    exponent = torch.where(amax > 0, exponent.clamp(min=-127), -127)
    scaled = torch.ldexp(v, -exponent)
    return torch.ldexp(scaled.to(torch.float8_e4m3fn).float(), exponent)


def _plain_rows(x):
    """One step per 128 consecutive elements of a row."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    return _plain_codes(v, v.abs().amax(-1, keepdim=True)).reshape(rows, -1)[:, :k]


def _plain_square(w):
    """One step per 128 x 128 elements."""
    n, k = w.shape
    v = torch.nn.functional.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK))
    v = v.reshape(-(-n // BLOCK), BLOCK, -(-k // BLOCK), BLOCK)
    v = _plain_codes(v, v.abs().amax((1, 3), keepdim=True))
    return v.reshape(-(-n // BLOCK) * BLOCK, -1)[:n, :k]


def _plain_linear(s, case):
    dtype = DTYPES[case["dtype"]]
    w = _plain_square(s["w"]) if case["train"] else s["weight8"]
    y = _plain_rows(s["x"]) @ w.t()
    y = (y if s["b"] is None else y + s["b"].float()).to(dtype)
    if not case["train"]:
        return y
    dy = s["grad"]
    out = {"y": y, "x": _plain_rows(dy) @ w,
           "w": _plain_rows(dy.t()) @ _plain_rows(s["x"].t()).t()}
    if s["b"] is not None:
        out["b"] = dy.float().sum(0)
    return {k: v.to(dtype) for k, v in out.items()}


def _plain_norm(v, kind):
    """(normalised v, 1 / deviation) in fp32."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * rstd, rstd


def _plain_angles(s):
    """cos and sin [.., tokens, rotated pairs] in fp32 (the angles need 64 bits),
    and the pairs' two members."""
    dims, interleaved = s["dims"], s["case"]["interleaved"]
    axis = torch.repeat_interleave(torch.arange(len(dims), device="cuda"),
                                   torch.tensor([d // 2 for d in dims], device="cuda"))
    size = torch.tensor(dims, device="cuda")[axis]
    start = (torch.cumsum(torch.tensor(dims, device="cuda"), 0)
             - torch.tensor(dims, device="cuda"))[axis]
    i = torch.arange(axis.numel(), device="cuda") - start // 2
    freq = BASE ** (-2.0 * i.double() / size)
    angle = s["pos"].clamp(min=0).double()[..., axis] * freq
    first = start + (2 * i if interleaved else i)
    second = first + 1 if interleaved else first + size // 2
    return torch.cos(angle).float(), torch.sin(angle).float(), first, second


def _plain_turn(t, angles, sign):
    """t [B, H, N, D] in fp32, each pair turned by its token's angle."""
    if angles is None:
        return t
    cos, sin, first, second = angles
    if cos.dim() == 3:  # positions of each sample
        cos, sin = cos[:, None], sin[:, None]
    u, v = t[..., first], t[..., second]
    out = t.clone()
    out[..., first] = u * cos - sign * v * sin
    out[..., second] = v * cos + sign * u * sin
    return out


def _plain_qkv(s, case):
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    b, n, _ = s["qkv"].shape
    angles = _plain_angles(s) if s["dims"] else None
    q, k, v = s["qkv"].reshape(b, n, h + 2 * hk, d).transpose(1, 2).split([h, hk, hk], 1)
    out = {}

    def side(name, t, dout):
        weight, bias = s[name + "_weight"].float(), s[name + "_bias"]
        normed, rstd = _plain_norm(t.float(), kind)
        value = normed * weight if bias is None else normed * weight + bias.float()
        out[name] = _plain_turn(value, angles, 1)
        if dout is None:
            return None
        dt = _plain_turn(dout.float(), angles, -1)
        out[name + "_weight"] = (dt * normed).sum((0, 1, 2))
        if bias is not None:
            out[name + "_bias"] = dt.sum((0, 1, 2))
        g = dt * weight
        back = g - normed * (g * normed).mean(-1, keepdim=True)
        if kind == "layer":
            back = back - g.mean(-1, keepdim=True)
        return back * rstd

    dq = side("q", q, s.get("grad_q"))
    dk = side("k", k, s.get("grad_k"))
    out["v"] = v.contiguous()
    if case["train"]:
        grad = torch.cat([dq, dk, s["grad_v"].float()], 1).transpose(1, 2)
        out["qkv"] = grad.reshape(b, n, -1)
    return {name: t.to(dtype) for name, t in out.items()}


def _plain_words(count, seed, offset):
    """The first `count` 32-bit words of Philox4x32-10 under a key and an upper
    counter half, as int64."""
    low = 0xFFFFFFFF
    i = torch.arange(-(-count // 4), device="cuda")
    c0, c1 = i & low, i >> 32
    c2, c3 = torch.full_like(i, offset & low), torch.full_like(i, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (64-bit products wrap; both halves are right)
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack([c0, c1, c2, c3], -1).reshape(-1)[:count]


def _draws(case):
    return {"element": (case["batch"], case["tokens"], case["dim"]),
            "row": (case["batch"], case["tokens"], 1), "sample": (case["batch"], 1, 1)}[case["per"]]


def _plain_dropout(s, case):
    dtype, p = DTYPES[case["dtype"]], case["p"]
    shape = _draws(case)
    words = _plain_words(math.prod(shape), s["seed"], s["offset"]).reshape(shape)
    keep = words >= int(round(p * 2.0 ** 32))
    scale = 1.0 / (1.0 - p)

    def masked(t):
        return torch.where(keep, t.float() * scale, 0.0)

    y = masked(s["x"])
    y = (y if s["residual"] is None else s["residual"].float() + y).to(dtype)
    if not case["train"]:
        return y
    out = {"y": y, "x": masked(s["grad"]).to(dtype)}
    if s["residual"] is not None:
        out["residual"] = s["grad"]
    return out


# ---------------------------------------------------------------- the package's calls

def _own_linear(s, case):
    from scmp_vit_b200 import fp8
    if not case["train"]:
        return fp8.fp8_matmul(s["x"], s["weight8"], bias=s["b"])
    y = fp8.fp8_linear(s["x"], s["w"], s["b"])
    names = [n for n in ("x", "w", "b") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["grad"])
    return {"y": y, **dict(zip(names, grads))}


def _own_qkv(s, case):
    from scmp_vit_b200.attention import split_qkv_norm
    q, k, v = split_qkv_norm(s["qkv"], case["heads"], s["q_weight"], s["k_weight"], s["q_bias"],
                             s["k_bias"], kind=case["kind"], eps=EPS, axes=s.get("axes"),
                             pos=s.get("pos"), num_kv_heads=case["kv_heads"], transpose_v=False)
    out = {"q": q, "k": k, "v": v}
    if case["train"]:
        names = [n for n in ("qkv", "q_weight", "k_weight", "q_bias", "k_bias")
                 if s[n] is not None]
        out.update(zip(names, torch.autograd.grad(
            (q, k, v), [s[n] for n in names], (s["grad_q"], s["grad_k"], s["grad_v"]))))
    return out


def _own_dropout(s, case):
    from scmp_vit_b200 import vit
    y = vit.dropout(s["x"], case["p"], s["seed"], s["offset"], per=case["per"],
                    residual=s["residual"])
    if not case["train"]:
        return y
    names = [n for n in ("x", "residual") if s[n] is not None]
    return {"y": y, **dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], s["grad"])))}


def run(state):
    case = state["case"]
    if own:
        return {"linear": _own_linear, "qkv": _own_qkv, "dropout": _own_dropout}[case["op"]](
            state, case)
    with torch.no_grad():
        return {"linear": _plain_linear, "qkv": _plain_qkv, "dropout": _plain_dropout}[
            case["op"]](state, case)


# ---------------------------------------------------------------- 64 bits, from the definitions

def _exact_grid():
    """The non-negative e4m3 numbers in order."""
    return torch.tensor([m * 2.0 ** -9 for m in range(8)] + [
        (8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:119],
        dtype=torch.float64, device="cuda")


def _exact_nearest(v, grid):
    """Nearest entry of a sorted grid, the even one between two."""
    border = (grid[1:] + grid[:-1]) / 2
    low = torch.searchsorted(border, v, right=False)  # borders below v
    high = torch.searchsorted(border, v, right=True)  # borders up to v
    return grid[torch.where((low != high) & (low % 2 == 1), high, low)]


def _exact_blocks(x, height, width):
    """The values of x's codes, one power of two per block of height x width: the
    smallest (from 2^-127 on) under which the block's largest is at most 448."""
    x = x.detach().double()
    rows, cols = x.shape
    out = torch.zeros(-(-rows // height) * height, -(-cols // width) * width,
                      dtype=torch.float64, device="cuda")
    out[:rows, :cols] = x
    v = out.view(out.shape[0] // height, height, out.shape[1] // width, width)
    top = v.abs().amax((1, 3), keepdim=True)
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -140))).clamp(min=-127)
    # log2 may round at a power of two: settle it by comparison
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 448 * torch.exp2(e - 1)) & (e > -127), e - 1, e)
    step = torch.exp2(e)
    q = _exact_nearest((v.abs() / step).contiguous(), _exact_grid())
    return (torch.sign(v) * q * step).view(out.shape)[:rows, :cols]


def _exact_linear(s, case):
    x = _exact_blocks(s["x"], 1, BLOCK)
    w = _exact_blocks(s["w"], BLOCK, BLOCK)
    bias = s["b"].detach().double() if s["b"] is not None else 0
    y = torch.einsum("mk,nk->mn", x, w) + bias
    if not case["train"]:
        return y
    del x
    out = {"y": y, "x": torch.einsum("mn,nk->mk", _exact_blocks(s["grad"], 1, BLOCK), w),
           "w": torch.einsum("mn,mk->nk", _exact_blocks(s["grad"], BLOCK, 1),
                             _exact_blocks(s["x"], BLOCK, 1))}
    if s["b"] is not None:
        out["b"] = s["grad"].double().sum(0)
    return out


def _exact_qkv(s, case):
    """Norms by their definition, gradients by the chain rule on centred rows, and
    each pair as a complex number, turned by e^(i angle)."""
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    b, n, _ = s["qkv"].shape
    x = s["qkv"].detach().double().reshape(b, n, h + 2 * hk, d).permute(0, 2, 1, 3)
    turn, order, base, at = None, [], 0, 0
    if s["dims"]:
        pos = s["pos"] if s["pos"].dim() == 3 else s["pos"][None]
        turn = torch.ones(pos.shape[0], 1, n, d // 2, dtype=torch.complex128, device="cuda")
        for a, da in enumerate(s["dims"]):
            for i in range(da // 2):
                angle = pos[..., a].double() * math.pow(BASE, -2.0 * i / da)
                angle = torch.where(pos[..., a] < 0, 0.0, angle)
                turn[:, 0, :, at] = torch.polar(torch.ones_like(angle), angle)
                order += [base + 2 * i, base + 2 * i + 1] if case["interleaved"] else [
                    base + i, base + i + da // 2]
                at += 1
            base += da
        order += list(range(base, d))
        order = torch.tensor(order, device="cuda")
        back = torch.argsort(order)

    def rotate(t, conj):
        if turn is None:
            return t
        c = torch.view_as_complex(t[..., order].reshape(*t.shape[:-1], d // 2, 2).contiguous())
        by = turn.conj() if conj else turn
        return torch.view_as_real(c * by).reshape(t.shape)[..., back]

    out, grads = {}, []
    for name, lo, count in (("q", 0, h), ("k", h, hk)):
        u = x[:, lo:lo + count]
        if case["kind"] == "layer":
            u = u - u.sum(-1, keepdim=True) / d
        dev = torch.sqrt((u ** 2).sum(-1, keepdim=True) / d + EPS)
        weight, bias = s[name + "_weight"].detach().double(), s[name + "_bias"]
        out[name] = rotate(u / dev * weight + (0 if bias is None else bias.detach().double()),
                           False)
        if case["train"]:
            dt = rotate(s["grad_" + name].double(), True)
            out[name + "_weight"] = torch.einsum("bhnd,bhnd->d", dt, u / dev)
            if bias is not None:
                out[name + "_bias"] = torch.einsum("bhnd->d", dt)
            gw = dt * weight
            du = gw / dev - u * (gw * u).sum(-1, keepdim=True) / (d * dev ** 3)
            if case["kind"] == "layer":
                du = du - du.sum(-1, keepdim=True) / d
            grads.append(du)
    out["v"] = x[:, h + hk:]
    if case["train"]:
        grads.append(s["grad_v"].double())
        out["qkv"] = torch.cat(grads, 1).permute(0, 2, 1, 3).reshape(b, n, -1)
    return out


def _exact_words(count, seed, offset):
    """Philox4x32-10 with every 64-bit product put together from 16-bit halves."""
    low = 0xFFFFFFFF

    def halves(m, c):
        a = (m & 0xFFFF) * c               # below 2^48
        b = (m >> 16) * c + (a >> 16)      # below 2^49
        return b >> 16, (b << 16 & low) | (a & 0xFFFF)

    i = torch.arange((count + 3) // 4, device="cuda")
    c = [i & low, i >> 32, i * 0 + (offset & low), i * 0 + (offset >> 32 & low)]
    for r in range(10):
        key = ((seed & low) + r * 0x9E3779B9 & low, (seed >> 32 & low) + r * 0xBB67AE85 & low)
        (h0, l0), (h1, l1) = halves(0xD2511F53, c[0]), halves(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
    return torch.stack(c, 1).flatten()[:count]


def _exact_dropout(s, case):
    shape = _draws(case)
    u = _exact_words(math.prod(shape), s["seed"], s["offset"]).reshape(shape).double()
    factor = (u >= round(case["p"] * 2.0 ** 32)).double() / (1 - case["p"])
    y = s["x"].detach().double() * factor
    y = y if s["residual"] is None else y + s["residual"].detach().double()
    if not case["train"]:
        return y
    out = {"y": y, "x": s["grad"].double() * factor}
    if s["residual"] is not None:
        out["residual"] = s["grad"].double()
    return out


@torch.no_grad()
def exact(case, seed):
    s = _raw(case, seed)
    return {"linear": _exact_linear, "qkv": _exact_qkv, "dropout": _exact_dropout}[case["op"]](
        s, case)
