"""The operators around a gated feed-forward half of a modulated transformer block, as measurable cases.

Three operators, each through the entry point that a user's program calls:

* ``gated``  ``ops.gated_linear``: both projections of a gated feed-forward, its activation and the product, alone or with
             the gradients of a training step
* ``norms``  ``ops.sandwich_norm``: the norm behind a block's half, its gate and residual scale, the residual sum, and the
             modulated norm ahead of the next half, alone or with their gradients
* ``w4``     ``ops.w4_linear``: products of a few rows with 4-bit weights and group scales (the modulation vectors)

Activations are N(0, 1) with one channel in a hundred scaled by 20, weights N(0, 0.02), modulation N(0, 0.1), incoming
gradients N(0, 1) for the norms and N(0, 0.05) for the gated projections, whose weights' sums over tokens stay in fp16's range.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
TILE_N, TILE_K = 16, 64  # a tile of packed 4-bit weights: 512 bytes
NIBBLES = (0, 2, 4, 6, 1, 3, 5, 7)  # the order of eight neighbouring weights in a 32-bit word


# ---------------------------------------------------------------------------------------------- cases


def _gated(name, m, k, f, dtype="bf16", act="silu", bias=False, train=False):
    return dict(name=name, kind="gated", m=m, k=k, f=f, dtype=dtype, act=act, bias=bias, train=train)


def _norms(name, batch, rows, c, dtype="bf16", norm="rms", weights=True, residual_scale=1.0, train=False):
    return dict(name=name, kind="norms", batch=batch, rows=rows, c=c, dtype=dtype, norm=norm, weights=weights, residual_scale=residual_scale, train=train)


def _w4(name, m, k, n, group=128, dtype="bf16", zeros=False, bias=True):
    return dict(name=name, kind="w4", m=m, k=k, n=n, group=group, dtype=dtype, zeros=zeros, bias=bias)


def listed():
    return [
        # one vector through a small model's gated projections (a pooled embedding): the weights' way from memory
        _gated("gated_one_row", 1, 1536, 8960),
        # a short prompt's text tokens, an odd number of them, in fp16 with the tanh form of GELU and biases
        _gated("gated_text_77", 77, 4096, 10240, "fp16", "gelu_tanh", True),
        # the small model's video at 480p and 81 frames: 32 760 tokens
        _gated("gated_small_480p", 32760, 1536, 8960),
        # a fine-tuning step on one picture with its prompt, ragged against every tile
        _gated("gated_train_picture", 1101, 1536, 4616, "fp16", "gelu_tanh", True, train=True),
        # a fine-tuning step of the large model's widths on 16 380 tokens
        _gated("gated_train_large", 16380, 5120, 13824, train=True),
        # one token between two halves of a block
        _norms("norms_one_row", 1, 1, 5120),
        # a cond / uncond pair of the small model at 480p, modulation per sample
        _norms("norms_small_480p_cfg", 2, 32760, 1536, residual_scale=0.5),
        # fine-tuning on three short clips: layer norms without weights, fp16, odd lengths
        _norms("norms_train_clips", 3, 777, 2056, "fp16", "layer", False, 0.25, train=True),
        # fine-tuning of the large model at 720p and 81 frames: 75 600 tokens
        _norms("norms_train_720p", 1, 75600, 5120, train=True),
        # the six modulation vectors of a large block from one timestep embedding
        _w4("w4_modulation_row", 1, 5120, 30720),
        # the same of a small block for a handful of timesteps: groups of 32 with zero points, fp16
        _w4("w4_modulation_rows", 5, 1536, 9216, 32, "fp16", True),
        # sixteen rows back to the small width, groups of 64, an odd number of outputs
        _w4("w4_sixteen_rows", 16, 8960, 1533, 64, "bf16", False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gated", "norms", "w4"))
    if kind == "w4":
        group = rng.choice((32, 64, 128))
        k = group * max(1, _log(rng, 256, 13824) // group)
        case = _w4("", _log(rng, 1, 16), k, _log(rng, 16, 30720), group, rng.choice(("bf16", "fp16")), rng.random() < 0.5, rng.random() < 0.5)
    elif kind == "norms":
        train = rng.random() < 0.5
        c, batch = 8 * _log(rng, 8, 640), rng.choice((1, 1, 2, 3, 5))
        rows = _log(rng, 1, max(1, min(75600, 75600 * 5120 // (c * batch))))
        case = _norms("", batch, rows, c, rng.choice(("bf16", "fp16")), rng.choice(("rms", "layer")), rng.random() < 0.5, rng.choice((1.0, 0.5, 0.125)), train)
    else:
        train = rng.random() < 0.5
        k, f = 8 * _log(rng, 16, 640), 8 * _log(rng, 16, 1728)
        most = 16380 * 5120 * 13824 // (k * f)
        m = _log(rng, 64 if train else 1, max(64, min(75600, most)))
        case = _gated("", m, k, f, rng.choice(("bf16", "fp16")), rng.choice(("silu", "gelu_tanh")), rng.random() < 0.5, train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs


def _activations(rows, c, dtype, g):
    """N(0, 1), one channel in a hundred scaled by 20."""
    x = torch.randn(rows, c, device="cuda", generator=g)
    x[:, ::100] *= 20
    return x.to(dtype)


def _normal(shape, std, dtype, g):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _pad(n, to):
    return -(-n // to) * to


def pack_w4(q):
    """Values 0 .. 15 [N, K] -> the packed weight [ceil(N / 16), ceil(K / 64), 512] uint8: tiles of 16 rows x 64 columns; 16 bytes for
    each (row mod 8, eight columns of a block of 32): its 32-bit words are (block 0, row), (block 0, row + 8), (block 1, row),
    (block 1, row + 8), the eight columns in each in the order NIBBLES, lowest bits first."""
    n, k = q.shape
    nt, kt = _pad(n, TILE_N) // TILE_N, _pad(k, TILE_K) // TILE_K
    full = torch.full((nt * TILE_N, kt * TILE_K), 8, dtype=torch.uint8, device=q.device)
    full[:n, :k] = q
    t = full.view(nt, 2, 8, kt, 2, 4, 8).permute(0, 3, 2, 5, 4, 1, 6)[..., list(NIBBLES)]
    return (t[..., 0::2] | (t[..., 1::2] << 4)).reshape(nt, kt, 512).contiguous()


def tile_groups(v):
    """[N, groups] -> [ceil(N / 16), groups, 16], zeros behind the last row."""
    n, groups = v.shape
    full = torch.zeros(_pad(n, TILE_N), groups, dtype=v.dtype, device=v.device)
    full[:n] = v
    return full.view(-1, TILE_N, groups).transpose(1, 2).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "gated":
        m, k, f, train = case["m"], case["k"], case["f"], case["train"]
        s["x"] = _activations(m, k, dtype, g)
        s["w_gate"], s["w_up"] = _normal((f, k), 0.02, dtype, g), _normal((f, k), 0.02, dtype, g)
        s["b_gate"] = _normal((f,), 0.5, dtype, g) if case["bias"] else None
        s["b_up"] = _normal((f,), 0.5, dtype, g) if case["bias"] else None
        leaves = [s[n] for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if s[n] is not None]
        if train:
            s["grad"] = _normal((m, f), 0.05, dtype, g)
    elif case["kind"] == "norms":
        b, rows, c, train = case["batch"], case["rows"], case["c"], case["train"]
        s["x"] = _activations(b * rows, c, dtype, g).view(b, rows, c)
        s["y"] = _activations(b * rows, c, dtype, g).view(b, rows, c)
        for n in ("gate", "scale", "shift"):
            s[n] = _normal((b, 1, c), 0.1, dtype, g)
        s["post_weight"] = 1 + _normal((c,), 0.1, torch.float32, g) if case["weights"] else None
        s["pre_weight"] = 1 + _normal((c,), 0.1, torch.float32, g) if case["weights"] else None
        leaves = [s[n] for n in ("x", "y", "gate", "scale", "shift", "post_weight", "pre_weight") if s[n] is not None]
        if train:
            s["grad_r"], s["grad_h"] = _normal((b, rows, c), 1.0, dtype, g), _normal((b, rows, c), 1.0, dtype, g)
    else:
        m, k, n, group = case["m"], case["k"], case["n"], case["group"]
        train, leaves = False, []
        s["x"] = _activations(m, k, dtype, g)
        w = (torch.randn(n, k, device="cuda", generator=g) * 0.02).view(n, k // group, group)
        if case["zeros"]:  # 0 .. 15 between a group's least and largest weight
            low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
            scale = ((high - low) / 15).clamp(min=1e-6).to(dtype)
            zero = torch.round(-low / scale.float()).clamp(0, 15)
        else:  # -8 .. 7 about zero
            scale = (w.abs().amax(-1) / 7).clamp(min=1e-6).to(dtype)
            zero = torch.full_like(scale, 8, dtype=torch.float32)
        q = torch.round(w / scale.float()[..., None] + zero[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
        s["weight"], s["weight_scale"] = pack_w4(q), tile_groups(scale)
        s["weight_zero"] = tile_groups(zero.to(torch.uint8)) if case["zeros"] else None
        s["bias"] = _normal((n,), 0.1, dtype, g) if case["bias"] else None
    if train:
        for t in leaves:
            t.requires_grad_(True)
        s["leaves"] = leaves
    return s


# ---------------------------------------------------------------------------------------------- the operators


def run(state):
    kind, train = state["case"]["kind"], state["case"].get("train", False)
    if own:
        return {"gated": _own_gated, "norms": _own_norms, "w4": _own_w4}[kind](state, train)
    with torch.no_grad():
        return {"gated": _plain_gated, "norms": _plain_norms, "w4": _plain_w4}[kind](state, train)


def _own_gated(s, train):
    from ksanadit_b200 import ops
    h = ops.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], act=s["case"]["act"])
    return [h, *torch.autograd.grad(h, s["leaves"], s["grad"])] if train else [h]


def _own_norms(s, train):
    from ksanadit_b200 import ops
    r, h = ops.sandwich_norm(s["x"], s["y"], gate=s["gate"], scale=s["scale"], shift=s["shift"], post_weight=s["post_weight"], pre_weight=s["pre_weight"],
                             residual_scale=s["case"]["residual_scale"], kind=s["case"]["norm"], eps=EPS)
    return [r, h, *torch.autograd.grad((r, h), s["leaves"], (s["grad_r"], s["grad_h"]))] if train else [r, h]


def _own_w4(s, train):
    from ksanadit_b200 import ops
    return [ops.w4_linear(s["x"], s["weight"], s["weight_scale"], s["weight_zero"], s["bias"], out_features=s["case"]["n"])]


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_gated(s, train):
    dtype = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.T, x @ wu.T
    if s["b_gate"] is not None:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    a, da = _activation(g, s["case"]["act"])
    out = [(a * u).to(dtype)]
    if train:
        d = s["grad"].float()
        dg, du = d * u * da, d * a
        out += [(dg @ wg + du @ wu).to(dtype), (dg.T @ x).to(dtype), (du.T @ x).to(dtype)]
        if s["b_gate"] is not None:
            out += [dg.sum(0).to(dtype), du.sum(0).to(dtype)]
    return out


def _standard(v, norm):
    """Rows of `v` normalised, and the factor of each row."""
    d = v - v.mean(-1, keepdim=True) if norm == "layer" else v
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    return d * rstd, rstd


def _standard_grad(d, n, rstd, norm):
    """The gradient of a normalised row's input from that of the row `n`."""
    e = d - n * (d * n).mean(-1, keepdim=True)
    return rstd * (e - d.mean(-1, keepdim=True) if norm == "layer" else e)


def _plain_norms(s, train):
    norm, scale_r, dtype = s["case"]["norm"], s["case"]["residual_scale"], s["x"].dtype
    x, y = s["x"].float(), s["y"].float()
    gate, scale, shift = s["gate"].float(), s["scale"].float(), s["shift"].float()
    wp, wn = (1.0, 1.0) if s["post_weight"] is None else (s["post_weight"], s["pre_weight"])
    yn, y_rstd = _standard(y, norm)
    r = x + scale_r * gate * (yn * wp)
    rn, r_rstd = _standard(r, norm)
    h = rn * wn * (1 + scale) + shift
    out = [r.to(dtype), h.to(dtype)]
    if train:
        dr, dh = s["grad_r"].float(), s["grad_h"].float()
        dr = dr + _standard_grad(dh * (1 + scale) * wn, rn, r_rstd, norm)
        dyn = scale_r * gate * dr
        out += [dr.to(dtype), _standard_grad(dyn * wp, yn, y_rstd, norm).to(dtype), (scale_r * dr * (yn * wp)).sum(1, keepdim=True).to(dtype),
                (dh * (rn * wn)).sum(1, keepdim=True).to(dtype), dh.sum(1, keepdim=True).to(dtype)]
        if s["post_weight"] is not None:
            out += [(dyn * yn).sum((0, 1)), (dh * (1 + scale) * rn).sum((0, 1))]
    return out


def _plain_w4(s, train):
    c = s["case"]
    n, k, nt, kt = c["n"], c["k"], s["weight"].shape[0], s["weight"].shape[1]
    b = s["weight"].view(nt, kt, 8, 4, 2, 2, 4)
    q = torch.stack([b & 15, b >> 4], -1).flatten(-2)  # eight columns in the order NIBBLES
    q = q[..., [0, 4, 1, 5, 2, 6, 3, 7]].permute(0, 5, 2, 1, 4, 3, 6).reshape(nt * TILE_N, kt * TILE_K)[:n, :k].float()
    scale = s["weight_scale"].float().transpose(1, 2).reshape(nt * TILE_N, -1)[:n, :, None]
    zero = 8.0 if s["weight_zero"] is None else s["weight_zero"].float().transpose(1, 2).reshape(nt * TILE_N, -1)[:n, :, None]
    w = ((q.view(n, k // c["group"], c["group"]) - zero) * scale).view(n, k)
    out = s["x"].float() @ w.T
    return [(out if s["bias"] is None else out + s["bias"].float()).to(s["x"].dtype)]


# ---------------------------------------------------------------------------------------------- what a pass needs


def work(case):
    if case["kind"] == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        b = 2 * (m * k + 2 * f * k + m * f + (2 * f if case["bias"] else 0))
        if case["train"]:  # the incoming gradient, and a gradient for each input
            b += 2 * (m * f + m * k + 2 * f * k + (2 * f if case["bias"] else 0))
        return {"bytes": b, "flops": (12 if case["train"] else 4) * m * k * f}
    if case["kind"] == "norms":
        m, c = case["batch"] * case["rows"], case["c"]
        b = 2 * 4 * m * c + 2 * 3 * case["batch"] * c + (8 * c if case["weights"] else 0)
        return {"bytes": 2 * b if case["train"] else b, "flops": (40 if case["train"] else 14) * m * c}
    m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
    b = n * k // 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * (k + n) + (2 * n if case["bias"] else 0)
    return {"bytes": b, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    wide = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor) and n not in ("weight", "weight_zero")}
    return {"gated": _exact_gated, "norms": _exact_norms, "w4": _exact_w4}[case["kind"]](case, s, wide)


def _exact_gated(case, s, w):
    names = [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if n in w]
    for n in names:
        w[n].requires_grad_(case["train"])
    g = torch.nn.functional.linear(w["x"], w["w_gate"], w.get("b_gate"))
    u = torch.nn.functional.linear(w["x"], w["w_up"], w.get("b_up"))
    h = (torch.nn.functional.silu(g) if case["act"] == "silu" else torch.nn.functional.gelu(g, approximate="tanh")) * u
    return [h.detach(), *torch.autograd.grad(h, [w[n] for n in names], w["grad"])] if case["train"] else [h]


def _exact_norms(case, s, w):
    names = [n for n in ("x", "y", "gate", "scale", "shift", "post_weight", "pre_weight") if n in w]
    for n in names:
        w[n].requires_grad_(case["train"])

    def norm(v, weight):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(v, (case["c"],), weight, None, EPS)
        return torch.nn.functional.rms_norm(v, (case["c"],), weight, EPS)

    r = w["x"] + case["residual_scale"] * w["gate"] * norm(w["y"], w.get("post_weight"))
    h = torch.addcmul(w["shift"], norm(r, w.get("pre_weight")), 1 + w["scale"])
    if not case["train"]:
        return [r, h]
    return [r.detach(), h.detach(), *torch.autograd.grad((r, h), [w[n] for n in names], (w["grad_r"], w["grad_h"]))]


def _exact_w4(case, s, w):
    # one product per weight of a tile: bytes to nibbles to places, by index
    n, k, device = case["n"], case["k"], s["weight"].device
    row, col = torch.arange(n, device=device)[:, None], torch.arange(k, device=device)[None, :]
    place = torch.tensor([NIBBLES.index(i) for i in range(8)], device=device)[col % 8]
    byte = ((row % 8) * 4 + (col % 32) // 8) * 16 + ((col % 64) // 32) * 8 + ((row % 16) // 8) * 4 + place // 2
    q = (s["weight"][row // TILE_N, col // TILE_K, byte] >> (4 * (place % 2)).to(torch.uint8)) & 15
    group = col // case["group"]
    zero = 8 if s["weight_zero"] is None else s["weight_zero"][row // TILE_N, group, row % TILE_N].double()
    full = (q.double() - zero) * w["weight_scale"][row // TILE_N, group, row % TILE_N]
    return [torch.nn.functional.linear(w["x"], full, w.get("bias"))]
