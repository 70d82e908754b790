"""The language-model operators of this framework, case by case: inputs, plain forms, exact values.

Three operators, each with the direction and the types it is used in:

* ``linear`` / ``quantise`` - matrix products in 8-bit floating point (e4m3) with one scale for
  each block of 128: activations in blocks of 1 x 128, weights in blocks of 128 x 128, forward and
  the gradient towards the activations;
* ``rotary`` / ``table`` - rotary positions: interleaved and half layouts, a part of the head, queries
  and keys together, gathered by position; cos/sin tables scaled for long contexts;
* ``group_norm`` - group normalisation with an activation over channels-last tensors, forward and
  backward.

``run`` computes the plain form in elementary torch operations, or, where ``own`` is true, calls the
framework's operators.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
E4M3_MAX = 448.0


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-zimage-triton_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import zimage_b200

    return zimage_b200


# --- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # one token through the fused query/key/value projection: latency, bound by the weight
        {"name": "linear_token", "op": "linear", "M": 1, "K": 3840, "N": 11520, "dtype": "bf16", "bias": False,
         "train": False},
        # a ragged prompt of caption features into the model width, with a bias, in fp16
        {"name": "linear_caption", "op": "linear", "M": 333, "K": 2560, "N": 3840, "dtype": "fp16", "bias": True,
         "train": False},
        # two guided images of 1024 x 1024: the projection over 18432 token rows
        {"name": "linear_image", "op": "linear", "M": 18432, "K": 3840, "N": 11520, "dtype": "bf16", "bias": False,
         "train": False},
        # an adapter trained through a frozen down projection: output, input gradient, bias gradient
        {"name": "linear_train", "op": "linear", "M": 4608, "K": 10240, "N": 3840, "dtype": "bf16", "bias": True,
         "train": True},
        # the activations of one guided image, quantised by rows
        {"name": "quantise_rows", "op": "quantise", "M": 9216, "K": 3840, "dtype": "bf16", "weight": False},
        # one new token for each of eight sequences at their own far positions
        {"name": "rotary_token", "op": "rotary", "B": 8, "S": 1, "H": 30, "Hk": 30, "D": 128, "R": 128, "L": 65536,
         "layout": "half", "dtype": "bf16", "gather": True, "fused": True, "train": False},
        # queries and keys of one guided image, slices of the fused projection
        {"name": "rotary_image", "op": "rotary", "B": 2, "S": 4608, "H": 30, "Hk": 30, "D": 128, "R": 128, "L": 4608,
         "layout": "interleaved", "dtype": "bf16", "gather": False, "fused": True, "train": False},
        # training on packed sequences: half of the head rotated, shared key heads, gradients
        {"name": "rotary_train", "op": "rotary", "B": 1, "S": 16383, "H": 24, "Hk": 6, "D": 128, "R": 64, "L": 16384,
         "layout": "half", "dtype": "bf16", "gather": True, "fused": False, "train": True},
        # the table of a context eight times the length trained on, scaled by parts
        {"name": "table_long", "op": "table", "T": 131072, "dim": 128, "theta": 10000.0, "scaling": "yarn",
         "factor": 8.0, "original": 16384},
        # a small odd latent: latency, ragged channels per group
        {"name": "group_norm_small", "op": "group_norm", "B": 1, "P": 391, "C": 96, "G": 32, "dtype": "fp16",
         "act": "silu", "affine": True, "train": False},
        # the inner level of a latent decoder, trained
        {"name": "group_norm_train", "op": "group_norm", "B": 2, "P": 16384, "C": 512, "G": 32, "dtype": "bf16",
         "act": "silu", "affine": True, "train": True},
        # the outer level of a latent decoder at 1024 x 1024
        {"name": "group_norm_image", "op": "group_norm", "B": 1, "P": 1048576, "C": 128, "G": 32, "dtype": "bf16",
         "act": "silu", "affine": True, "train": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "quantise", "rotary", "rotary", "table", "group_norm", "group_norm"])
    if op == "linear":
        train = rng.random() < 0.35
        K, N = _spread(rng, 96, 10240), _spread(rng, 96, 11520)
        if rng.random() < 0.6:  # most widths are whole blocks
            K, N = -(-K // BLOCK) * BLOCK, -(-N // BLOCK) * BLOCK
        most = 18432 * 3840 * 11520 // (2 if train else 1)
        return {"op": op, "M": min(_spread(rng, 1, 18432), max(1, most // (K * N))), "K": K, "N": N,
                "dtype": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.5, "train": train}
    if op == "quantise":
        K = _spread(rng, 64, 10240)
        if rng.random() < 0.6:
            K = -(-K // BLOCK) * BLOCK
        return {"op": op, "M": _spread(rng, 1, 18432), "K": K, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "weight": rng.random() < 0.4}
    if op == "rotary":
        D = rng.choice([32, 48, 64, 80, 96, 128, 192, 256])
        R = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        B, S, H = rng.choice([1, 1, 2, 3, 8]), _spread(rng, 1, 16384), _spread(rng, 1, 32)
        S = max(1, min(S, 2 * 4608 * 30 * 128 // (B * H * D)))
        gather = rng.random() < 0.6
        return {"op": op, "B": B, "S": S, "H": H, "Hk": rng.choice([0, 1, H, max(1, H // 4)]), "D": D, "R": R,
                "L": S if not gather else max(S, _spread(rng, 64, 131072)),
                "layout": rng.choice(["interleaved", "half"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "gather": gather, "fused": rng.random() < 0.5, "train": rng.random() < 0.4}
    if op == "table":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": op, "T": _spread(rng, 64, 131072), "dim": 2 * rng.randint(16, 64),
                "theta": rng.choice([256.0, 10000.0, 500000.0]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else round(rng.uniform(1.5, 16.0), 2),
                "original": _spread(rng, 1024, 32768)}
    G = rng.choice([1, 4, 8, 16, 32, 32])
    C = G * _spread(rng, 1, 1024 // G)
    B = rng.choice([1, 1, 2, 4])
    train = rng.random() < 0.4
    most = 1048576 * 128 // (B * C * (3 if train else 1))
    least = -(-16 * G // C) if train else 1  # a gradient through a handful of values says little
    return {"op": op, "B": B, "P": max(least, min(_spread(rng, 1, 1048576), max(1, most))), "C": C, "G": G,
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "act": rng.choice(["silu", "silu", "none"]),
            "affine": rng.random() < 0.8, "train": train}


# --- inputs -----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, M, K, dtype):
    """Unit normal rows with one channel in a hundred twenty times as large."""
    x = _normal(g, M, K)
    x *= torch.where(torch.rand(K, generator=g, device="cuda") < 0.01, 20.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": case}
    if op == "linear":
        dt, M, K, N = DTYPES[case["dtype"]], case["M"], case["K"], case["N"]
        st["x"] = _activations(g, M, K, dt).requires_grad_(case["train"])
        w = (_normal(g, N, K) * (1.0 / math.sqrt(K))).to(torch.bfloat16)
        st["wq"], st["ws"] = _weight_blocks(w)
        st["bias"] = None
        if case["bias"]:
            st["bias"] = (_normal(g, N) * 0.5).to(dt).requires_grad_(case["train"])
        if case["train"]:
            st["wqt"] = st["wq"].t().contiguous()
            st["dy"] = (_normal(g, M, N) * 1e-3).to(dt)
        return st
    if op == "quantise":
        dt, M, K = DTYPES[case["dtype"]], case["M"], case["K"]
        st["x"] = (_normal(g, M, K) * 0.02).to(dt) if case["weight"] else _activations(g, M, K, dt)
        return st
    if op == "rotary":
        dt, B, S, H, Hk, D = DTYPES[case["dtype"]], case["B"], case["S"], case["H"], case["Hk"], case["D"]
        R, L = case["R"], case["L"]
        if case["fused"]:  # slices of one projection: queries, keys, values
            qkv = _normal(g, B, S, (H + 2 * Hk) * D).to(dt)
            q = qkv[..., :H * D].unflatten(-1, (H, D))
            k = qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)) if Hk else None
        else:
            q = _normal(g, B, S, H, D).to(dt)
            k = _normal(g, B, S, Hk, D).to(dt) if Hk else None
        st["q"], st["k"] = q.detach().requires_grad_(case["train"]), None
        if k is not None:
            st["k"] = k.detach().requires_grad_(case["train"])
        pos = torch.arange(L, device="cuda", dtype=torch.float64)
        freq = torch.exp(torch.arange(R // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(10000.0) / R))
        ang = pos[:, None] * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["positions"] = None
        if case["gather"]:  # each row's own start, as sequences of a batch have
            start = torch.randint(0, L - S + 1, (B, 1), generator=g, device="cuda")
            st["positions"] = start + torch.arange(S, device="cuda")
        if case["train"]:
            st["dq"] = _normal(g, B, S, H, D).to(dt)
            st["dk"] = _normal(g, B, S, Hk, D).to(dt) if Hk else None
        return st
    if op == "table":
        start = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
        st["positions"] = torch.arange(start, start + case["T"], device="cuda")
        return st
    dt, B, P, C = DTYPES[case["dtype"]], case["B"], case["P"], case["C"]
    # every channel with a mean and a spread of its own
    x = _normal(g, B, P, C)
    x *= 0.5 + torch.rand(C, generator=g, device="cuda")
    x += _normal(g, C)
    st["x"] = x.to(dt).requires_grad_(case["train"])
    st["w"] = st["b"] = None
    if case["affine"]:
        st["w"] = (1.0 + 0.1 * _normal(g, C)).requires_grad_(case["train"])
        st["b"] = (0.1 * _normal(g, C)).requires_grad_(case["train"])
    if case["train"]:
        st["dy"] = _normal(g, B, P, C).to(dt)
    return st


# --- plain forms ------------------------------------------------------------------------------


def _pow2_scale(amax):
    """The smallest power of two s (at least 2^-120) with amax <= 448 s; NaN where amax is not finite."""
    mant, expo = torch.frexp(amax)  # amax = mant 2^expo, mant in [1/2, 1); 448 = 0.875 * 2^9
    e = (expo - 9 + (mant > 0.875).to(expo.dtype)).clamp(min=-120)
    s = torch.ldexp(torch.ones_like(amax), e)
    s = torch.where(amax == 0, torch.full_like(s, 2.0 ** -120), s)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


def _row_blocks(x):
    """e4m3 values of x [M, K] in blocks of 1 x 128, and the blocks' scales [M, ceil(K / 128)]."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    xf = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K)).view(M, kb, BLOCK)
    s = _pow2_scale(xf.abs().amax(-1))
    q = (xf / s[..., None]).to(torch.float8_e4m3fn).view(M, kb * BLOCK)[:, :K]
    return q, s


def _weight_blocks(w):
    """e4m3 values of w [N, K] in blocks of 128 x 128, and the blocks' scales."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    wf = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    s = _pow2_scale(wf.abs().amax((1, 3)))
    q = (wf / s[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.contiguous(), s


def _spread_rows(q, s):
    """q [M, K] times its scales [M, ceil(K / 128)]."""
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _spread_blocks(q, s):
    """q [N, K] times its scales [ceil(N / 128), ceil(K / 128)]."""
    return q.float() * s.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _turn(x, cos, sin, layout):
    """x [B, S, H, D] with its first 2 * cos.shape[-1] features rotated."""
    half = cos.shape[-1]
    xf = x.float()
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if layout == "half":
        a, b = xf[..., :half], xf[..., half:2 * half]
        rot = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        rot = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([rot, xf[..., 2 * half:]], -1).to(x.dtype)


def _frequencies(case, device):
    dim, theta, factor = case["dim"], case["theta"], case["factor"]
    j = torch.arange(dim // 2, device=device, dtype=torch.float64)
    if case["scaling"] == "ntk":
        theta = theta * factor ** (dim / (dim - 2))
    f = torch.exp(j * (-2.0 * math.log(theta) / dim))
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":
        turns = case["original"] * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = (1.0 - keep) * f / factor + keep * f
    return f, (0.1 * math.log(factor) + 1.0 if case["scaling"] == "yarn" else 1.0)


def _plain_group_norm(st):
    case = st["case"]
    x, C, G = st["x"].detach(), case["C"], case["G"]
    B, P, cpg = case["B"], case["P"], case["C"] // case["G"]
    xf = x.float()
    mean = xf.view(B, P, G, cpg).mean((1, 3))
    cen = xf - mean.repeat_interleave(cpg, 1)[:, None]
    rstd = torch.rsqrt(cen.square().view(B, P, G, cpg).mean((1, 3)) + 1e-6)
    xhat = cen * rstd.repeat_interleave(cpg, 1)[:, None]
    z = xhat
    if st["w"] is not None:
        z = xhat * st["w"].detach() + st["b"].detach()
    sig = torch.sigmoid(z) if case["act"] == "silu" else None
    y = (z * sig if sig is not None else z).to(x.dtype)
    if not case["train"]:
        return y
    gz = st["dy"].float()
    if sig is not None:
        gz = gz * (sig * (1.0 + z * (1.0 - sig)))
    db, dw = gz.sum((0, 1)), (gz * xhat).sum((0, 1))
    if st["w"] is not None:
        gz = gz * st["w"].detach()
    c1 = gz.view(B, P, G, cpg).mean((1, 3)).repeat_interleave(cpg, 1)[:, None]
    c2 = (gz * xhat).view(B, P, G, cpg).mean((1, 3)).repeat_interleave(cpg, 1)[:, None]
    dx = ((gz - c1 - xhat * c2) * rstd.repeat_interleave(cpg, 1)[:, None]).to(x.dtype)
    return [y, dx] + ([dw, db] if st["w"] is not None else [])


def _plain(st):
    case = st["case"]
    op = case["op"]
    if op == "linear":
        x = st["x"].detach()
        w = _spread_blocks(st["wq"], st["ws"])
        y = _spread_rows(*_row_blocks(x)) @ w.t()
        if st["bias"] is not None:
            y = y + st["bias"].detach().float()
        y = y.to(x.dtype)
        if not case["train"]:
            return y
        dx = (_spread_rows(*_row_blocks(st["dy"])) @ w).to(x.dtype)
        out = [y, dx]
        if st["bias"] is not None:
            out.append(st["dy"].float().sum(0).to(x.dtype))
        return out
    if op == "quantise":
        q, s = _weight_blocks(st["x"]) if case["weight"] else _row_blocks(st["x"])
        return [q.float(), s]
    if op == "rotary":
        if st["positions"] is not None:
            cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
        else:
            cos, sin = st["cos"][:case["S"]], st["sin"][:case["S"]]
        out = [_turn(t.detach(), cos, sin, case["layout"]) for t in (st["q"], st["k"]) if t is not None]
        if case["train"]:
            out += [_turn(t, cos, -sin, case["layout"]) for t in (st["dq"], st["dk"]) if t is not None]
        return out
    if op == "table":
        f, m = _frequencies(case, "cuda")
        ang = st["positions"].double()[:, None] * f
        return [(ang.cos() * m).float(), (ang.sin() * m).float()]
    return _plain_group_norm(st)


# --- the framework's operators ----------------------------------------------------------------


def _own(st):
    z = _ops()
    case = st["case"]
    op = case["op"]
    if op == "linear":
        y = z.fp8_block_linear(st["x"], st["wq"], st["ws"], st["bias"], w_q_t=st.get("wqt"))
        if not case["train"]:
            return y
        leaves = [st["x"]] + ([st["bias"]] if st["bias"] is not None else [])
        return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]
    if op == "quantise":
        q, s = (z.fp8_block_quantize_weight if case["weight"] else z.fp8_block_quantize)(st["x"])
        return [q.float(), s]
    if op == "rotary":
        q, k = z.rotary_embed(st["q"], st["k"], st["cos"], st["sin"], positions=st["positions"],
                              layout=case["layout"])
        out = [t for t in (q, k) if t is not None]
        if not case["train"]:
            return out
        leaves, grads = [st["q"]], [st["dq"]]
        if k is not None:
            leaves, grads = leaves + [st["k"]], grads + [st["dk"]]
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))
    if op == "table":
        scaling = None
        if case["scaling"] != "none":
            scaling = {"type": case["scaling"], "factor": case["factor"], "original_length": case["original"]}
        return list(z.rotary_table(st["positions"], case["dim"], theta=case["theta"], scaling=scaling))
    y = z.group_norm_act(st["x"], case["G"], st["w"], st["b"], eps=1e-6, activation=case["act"])
    if not case["train"]:
        return y
    leaves = [st["x"]] + ([st["w"], st["b"]] if st["w"] is not None else [])
    return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]


def run(state):
    return _own(state) if own else _plain(state)


# --- what a pass cannot do without ------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "linear":
        M, K, N, train = case["M"], case["K"], case["N"], case["train"]
        blocks = -(-N // BLOCK) * -(-K // BLOCK)
        b = M * K * 2 + N * K + 4 * blocks + M * N * 2 + (2 * N if case["bias"] else 0)
        if train:
            b += M * N * 2 + M * K * 2 + (2 * N if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * M * N * K * (2 if train else 1)}
    if op == "quantise":
        M, K, kb = case["M"], case["K"], -(-case["K"] // BLOCK)
        size = 4 if case["dtype"] == "fp32" else 2
        scales = -(-M // BLOCK) * kb if case["weight"] else M * kb
        return {"bytes": M * K * (size + 1) + 4 * scales, "flops": 2 * M * K}
    size = 4 if case.get("dtype") == "fp32" else 2
    if op == "rotary":
        n = case["B"] * case["S"] * (case["H"] + case["Hk"]) * case["D"] * (2 if case["train"] else 1)
        rows = min(case["L"], case["B"] * case["S"]) if case["gather"] else case["S"]
        return {"bytes": 2 * n * size + rows * case["R"] * 4 + (8 * case["B"] * case["S"] if case["gather"] else 0),
                "flops": 3 * n}
    if op == "table":
        return {"bytes": case["T"] * (8 + case["dim"] * 4), "flops": case["T"] * case["dim"] * 4}
    n = case["B"] * case["P"] * case["C"]
    # forward: x in, y out; backward: x, dy in, dx out
    return {"bytes": n * size * (5 if case["train"] else 2) + 16 * case["C"], "flops": n * (30 if case["train"] else 12)}


# --- exact values, in 64 bits -----------------------------------------------------------------


def _exact_scale(amax):
    """2^e with the least e >= -120 such that amax / 2^e <= 448, found by trying."""
    e = torch.ceil(torch.log2(torch.clamp(amax, min=2.0 ** -140) / E4M3_MAX))
    e = torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)
    return torch.exp2(e.clamp(min=-120.0))


def _exact_e4m3(v):
    """v rounded to the nearest e4m3 value, ties to the even one: steps of 2^(e-3), never below 2^-9."""
    e = torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.clamp(torch.round(v / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_rows(x):
    """(values on the e4m3 grid, scales) by rows, block after block of columns."""
    v, s = torch.empty(x.shape, dtype=torch.float64, device=x.device), []
    for k0 in range(0, x.shape[1], BLOCK):
        part = x[:, k0:k0 + BLOCK].double()
        sc = _exact_scale(part.abs().max(1, keepdim=True).values)
        v[:, k0:k0 + BLOCK] = _exact_e4m3(part / sc)
        s.append(sc)
    return v, torch.cat(s, 1)


def _exact_product(xv, xs, w):
    """sum over blocks of (xv_b xs_b) w_b^T, w [N, K] in 64 bits."""
    y = torch.zeros(xv.shape[0], w.shape[0], dtype=torch.float64, device=xv.device)
    for b in range(xs.shape[1]):
        k0 = b * BLOCK
        y += (xv[:, k0:k0 + BLOCK] * xs[:, b:b + 1]) @ w[:, k0:k0 + BLOCK].t()
    return y


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "linear":
            w = st["wq"].double()
            for i in range(st["ws"].shape[0]):
                for j in range(st["ws"].shape[1]):
                    w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= st["ws"][i, j].double()
            y = _exact_product(*_exact_rows(st["x"]), w)
            if st["bias"] is not None:
                y += st["bias"].double()
            if not case["train"]:
                return y
            out = [y, _exact_product(*_exact_rows(st["dy"]), w.t().contiguous())]
            return out + ([st["dy"].double().sum(0)] if st["bias"] is not None else [])
        if op == "quantise":
            if not case["weight"]:
                return list(_exact_rows(st["x"]))
            x = st["x"].double()
            M, K = x.shape
            v, s = torch.empty_like(x), x.new_empty(-(-M // BLOCK), -(-K // BLOCK))
            for i in range(s.shape[0]):
                for j in range(s.shape[1]):
                    at = (slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
                    s[i, j] = _exact_scale(x[at].abs().max())
                    v[at] = _exact_e4m3(x[at] / s[i, j])
            return [v, s]
        if op == "rotary":
            B, S, half = case["B"], case["S"], case["R"] // 2
            pos = st["positions"]
            if pos is None:
                pos = torch.arange(S, device="cuda").expand(B, S)
            z = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, :, None]

            def turned(t, z):
                v = t.double().clone()
                at = [slice(0, half), slice(half, 2 * half)]
                if case["layout"] == "interleaved":
                    at = [slice(0, 2 * half, 2), slice(1, 2 * half, 2)]
                r = torch.complex(v[..., at[0]].contiguous(), v[..., at[1]].contiguous()) * z
                v[..., at[0]], v[..., at[1]] = r.real, r.imag
                return v

            out = [turned(t, z) for t in (st["q"], st["k"]) if t is not None]
            if case["train"]:
                out += [turned(t, z.conj()) for t in (st["dq"], st["dk"]) if t is not None]
            return out
        if op == "table":
            dim, fac, theta, L = case["dim"], case["factor"], case["theta"], case["original"]
            cols, m = [], 1.0
            for j in range(dim // 2):
                f = theta ** (-2.0 * j / dim)
                if case["scaling"] == "linear":
                    f /= fac
                elif case["scaling"] == "ntk":
                    f = (theta * fac ** (dim / (dim - 2.0))) ** (-2.0 * j / dim)
                elif case["scaling"] == "yarn":
                    ramp = min(1.0, max(0.0, (L * f / (2 * math.pi) - 1.0) / 31.0))
                    f = f / fac + ramp * (f - f / fac)
                    m = 1.0 + math.log(fac) / 10.0
                cols.append(f)
            ang = torch.outer(st["positions"].double(), torch.tensor(cols, dtype=torch.float64, device="cuda"))
            return [m * torch.cos(ang), m * torch.sin(ang)]
        B, P, C, G = case["B"], case["P"], case["C"], case["G"]
        x = st["x"].double().view(B, P, G, C // G)
        var, mean = torch.var_mean(x, dim=(1, 3), keepdim=True, correction=0)
        r = 1.0 / torch.sqrt(var + 1e-6)
        h = (x - mean) * r
        w = st["w"].double().view(G, -1) if st["w"] is not None else torch.ones(G, C // G, dtype=x.dtype, device=x.device)
        b = st["b"].double().view(G, -1) if st["b"] is not None else torch.zeros_like(w)
        z = h * w + b
        e = 1.0 / (1.0 + torch.exp(-z))
        y = z * e if case["act"] == "silu" else z
        if not case["train"]:
            return y.view(B, P, C)
        d = st["dy"].double().view_as(x)
        if case["act"] == "silu":
            d = d * (e + y * (1.0 - e))
        dw, db = (d * h).sum((0, 1)).view(C), d.sum((0, 1)).view(C)
        d = d * w
        dx = r * (d - d.mean((1, 3), keepdim=True) - h * (d * h).mean((1, 3), keepdim=True))
        return [y.view(B, P, C), dx.view(B, P, C)] + ([dw, db] if st["w"] is not None else [])
