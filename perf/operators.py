"""The operators around the attention inputs of a QLoRA step, as cases to be timed and compared:

- ``dropout``: dropout from a counter-based generator (``ops.dropout``), alone or added to a residual;
- ``lora``: the LoRA down projections of one input under such dropout, one mask for each branch, and
  their backward pass (``ops.lora_down_dropout``, ``ops.lora_down_dropout_bwd``);
- ``norm``: the norm of each query and key head with the position rotation from tables of cosines
  and sines (``ops.qk_norm_rope_fwd``, ``ops.qk_norm_rope_bwd``);
- ``axes``: the rotation by positions of several axes (time, height, width), with or without those
  norms (``ops.rope_axes_fwd``, ``ops.rope_axes_bwd``).

The mask of the generator: the value at index i of a row-major tensor is kept where its 16 random
bits are at least round(p * 65536). They are the (i % 8)-th 16 bits (low half of a word first) of
Philox4x32 with 7 rounds (Salmon et al., SC 2011), key = the 64-bit seed, counter = (i // 8, offset
+ stream), both 64-bit. A kept value is multiplied by 65536 / (65536 - round(p * 65536)).
"""

import math

import numpy as np
import torch

own = False

M32 = 0xFFFFFFFF
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # serving: one step of 8 running sequences of the 1.5B shape; launch latency counts
        dict(name="norm fwd 8 tokens", op="norm", bwd=False, tokens=8, heads=12, kv=2, dim=128, rot=128,
             dtype="bf16", lora=False),
        # the packed long-context batch of the 7B shape (131,072 tokens, 28 / 4 heads)
        dict(name="norm fwd 131072 tokens", op="norm", bwd=False, tokens=131072, heads=28, kv=4, dim=128, rot=128,
             dtype="bf16", lora=False),
        # a ragged fp16 batch with the LoRA delta of the queries and a part of the head rotated
        dict(name="norm fwd ragged, lora, part rotated", op="norm", bwd=False, tokens=4099, heads=14, kv=2, dim=80,
             rot=48, dtype="fp16", lora=True),
        # the training step of the 1.5B shape: 16,384 packed tokens
        dict(name="norm bwd 16384 tokens", op="norm", bwd=True, tokens=16384, heads=12, kv=2, dim=128, rot=128,
             dtype="bf16", lora=False),
        # one new token of one sequence, without norms
        dict(name="axes fwd 1 token", op="axes", bwd=False, tokens=1, heads=28, kv=4, dim=128, rot=128, dtype="bf16",
             axes=3, inter=False, norm=False, far=100000),
        # images among text, three axes, the training step's 16,384 tokens
        dict(name="axes fwd 16384 tokens", op="axes", bwd=False, tokens=16384, heads=12, kv=2, dim=128, rot=128,
             dtype="bf16", axes=3, inter=False, norm=False, far=4096),
        # the same with the norms and interleaved sections, a ragged length, far positions: backward
        dict(name="axes and norm bwd ragged", op="axes", bwd=True, tokens=10007, heads=16, kv=4, dim=64, rot=64,
             dtype="bf16", axes=3, inter=True, norm=True, far=1000000),
        # the config of 830 packed tokens: the gradient through a dropout
        dict(name="dropout 830 tokens", op="dropout", rows=830, width=1536, dtype="fp16", res="", p=0.1),
        # a layer's branch added to the residual stream of the training step
        dict(name="dropout and residual 16384 tokens", op="dropout", rows=16384, width=1536, dtype="bf16", res="fp32",
             p=0.05),
        # q and v LoRA, rank 16, of the 830-token config and of the training step, and its backward
        dict(name="lora fwd 830 tokens", op="lora", bwd=False, rows=830, width=1536, rank=16, branches=2, x="fp32",
             dtype="bf16", p=0.05),
        dict(name="lora fwd 16384 tokens", op="lora", bwd=False, rows=16384, width=1536, rank=16, branches=2, x="fp32",
             dtype="bf16", p=0.05),
        dict(name="lora bwd 16384 tokens", op="lora", bwd=True, rows=16384, width=1536, rank=16, branches=2, x="fp32",
             dtype="bf16", p=0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "axes", "dropout", "lora"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "dropout":
        rows, width = _log(rng, 1, 20000), _log(rng, 7, 3584)
        return dict(op=op, rows=rows, width=width, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    res=rng.choice(["", "fp32"]), p=rng.choice([0.0, 0.05, 0.1, 0.25, round(rng.uniform(0.01, 0.9), 3)]))
    if op == "lora":
        branches = rng.choice([1, 2])
        rank = rng.choice([8, 16, 24, 32] + ([64] if branches == 1 else []))
        return dict(op=op, bwd=rng.random() < 0.5, rows=_log(rng, 1, 16384), width=8 * _log(rng, 8, 450), rank=rank,
                    branches=branches, x=rng.choice(["fp32", "same"]), dtype=dtype,
                    p=rng.choice([0.05, 0.1, round(rng.uniform(0.01, 0.6), 3)]))
    dim = rng.choice([64, 80, 96, 128, 256])
    rot = dim if rng.random() < 0.7 else 16 * max(1, dim // 32)
    kv = rng.choice([1, 2, 3, 4, 8])
    case = dict(op=op, bwd=rng.random() < 0.5, tokens=_log(rng, 1, 24000), heads=kv * rng.choice([1, 2, 5, 7]), kv=kv,
                dim=dim, rot=rot, dtype=dtype)
    if op == "norm":
        return dict(case, lora=rng.random() < 0.3)
    return dict(case, axes=rng.choice([1, 2, 3, 4]), inter=rng.random() < 0.5, norm=rng.random() < 0.5,
                far=_log(rng, 64, 2000000))


def _sections(rot, axes):
    """rot / 2 frequencies shared out over the axes, the first (time) taking what is left."""
    n = rot // 2
    part = n // (axes + 1) if axes > 1 else 0
    return (n - part * (axes - 1),) + (part,) * (axes - 1)


def work(case):
    e = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "dropout":
        n = case["rows"] * case["width"]
        out = e[case["res"] or case["dtype"]]
        return {"bytes": n * (e[case["dtype"]] + (out if case["res"] else 0) + out), "flops": 2 * n}
    if case["op"] == "lora":
        n, r = case["rows"] * case["width"], case["rank"] * case["branches"]
        if case["bwd"]:  # du, x16, the addend and A in; dx and dA out
            return {"bytes": n * (2 + 4 + 4) + case["rows"] * r * 2 + r * case["width"] * (2 + 4), "flops": 4 * n * r}
        x = 4 + 2 if case["x"] == "fp32" else 2
        return {"bytes": n * x + case["rows"] * r * 2 + r * case["width"] * 2, "flops": 2 * n * r}
    t, d = case["tokens"], case["dim"]
    q, k = t * case["heads"] * d * 2, t * case["kv"] * d * 2
    normed = case["op"] == "norm" or case["norm"]
    b = 2 * (q + k)
    if case["bwd"] and normed:
        b += q + k
    if case.get("lora"):
        b += q
    b += 2 * t * case["rot"] * 4 if case["op"] == "norm" else case["axes"] * t * 8
    return {"bytes": b, "flops": (q + k) // 2 * (12 if case["bwd"] else 6)}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _positions(tokens, axes, far, g):
    """int64 [axes, tokens]: runs of text (all axes alike) and of grids (the first axis stands, the
    others walk over a grid), from a start up to ``far``."""
    i = torch.arange(tokens, device="cuda")
    start = torch.randint(max(1, far // 2), far + 1, (1,), generator=g, device="cuda")
    side = 24
    grid = (i // (side * side)) % 2 == 1
    base = start + (i // (side * side)) * side
    text = start + i
    walk = [base, base + (i // side) % side, base + i % side, base + (i * 7) % 5]
    return torch.stack([torch.where(grid, w, text) for w in walk[:axes]])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    randn = lambda *s, dt=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=dt)
    s = dict(case=case)
    dt = DT[case["dtype"]]
    if case["op"] in ("dropout", "lora"):
        # (seed, offset) of the step, on the device; the offset is past 32 bits for some seeds
        s["rng"] = torch.tensor([(seed + 1) * 0x9E3779B97F4A7C1 % (1 << 63), (seed % 3) * (1 << 32) + 4 * seed], device="cuda")
        s["stream"] = 2 * (seed % 28)
    if case["op"] == "dropout":
        s["x"] = randn(case["rows"], case["width"], dt=dt)
        s["residual"] = randn(case["rows"], case["width"], dt=DT[case["res"]]) if case["res"] else None
        return s
    if case["op"] == "lora":
        rows, width, r = case["rows"], case["width"], case["rank"] * case["branches"]
        # lora_A as its usual initialisation leaves it, the norm's output as input
        s["a"] = ((torch.rand(r, width, generator=g, device="cuda") * 2 - 1) / math.sqrt(width)).to(dt)
        s["p"] = (case["p"], case["p"] / 2)[:case["branches"]]
        if case["bwd"]:
            s["x"] = randn(rows, width, dt=dt)
            s["du"] = (randn(rows, r) * 0.05).to(dt)
            s["addend"] = randn(rows, width) * 0.05
        else:
            s["x"] = randn(rows, width, dt=torch.float32 if case["x"] == "fp32" else dt)
        return s
    t, h, kv, d, rot = (case[n] for n in ("tokens", "heads", "kv", "dim", "rot"))
    # queries and keys as slices of one projection's output, with a common offset as a bias gives
    if t * (h + 2 * kv) * d < 1 << 31:
        proj = randn(t, h + 2 * kv, d, dt=dt) + randn(h + 2 * kv, d, dt=dt)
        s["q"], s["k"] = proj[:, :h], proj[:, h:h + kv]
    else:
        s["q"], s["k"] = randn(t, h, d, dt=dt), randn(t, kv, d, dt=dt)
    normed = case["op"] == "norm" or case["norm"]
    s["eps"] = 1e-6
    s["wq"] = 1 + 0.2 * randn(d) if normed else None
    s["wk"] = 1 + 0.2 * randn(d) if normed else None
    s["lora"] = randn(t, h, d, dt=dt) * 0.1 if case.get("lora") else None
    inv = (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)).float()
    if case["op"] == "norm":
        ang = torch.arange(t, device="cuda")[:, None].double() * inv.double()
        ang = torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        s["inv"], s["sections"] = inv, _sections(rot, case["axes"])
        s["positions"] = _positions(t, case["axes"], case["far"], g)
    if case["bwd"]:
        s["gq"], s["gk"] = randn(h, t, d, dt=dt), randn(kv, t, d, dt=dt)
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _keep(rows, width, p, rng, stream):
    """(keep [rows, width], scale) of one stream of the generator."""
    n = rows * width
    i = torch.arange(-(-n // 8), device=rng.device)
    off = rng[1] + stream
    c0, c1, c2, c3 = i & M32, i >> 32, off & M32, (off >> 32) & M32
    k0, k1 = rng[0] & M32, (rng[0] >> 32) & M32
    for _ in range(7):  # the generator's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    bits = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)
    cut = math.floor(p * 65536 + 0.5)
    return (bits.reshape(-1)[:n] >= cut).view(rows, width), 65536 / (65536 - cut)


def _plain_dropout(s):
    c, x = s["case"], s["x"]
    keep, scale = _keep(c["rows"], c["width"], c["p"], s["rng"], s["stream"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        return s["residual"] + y
    return y.to(x.dtype)


def _plain_lora(s):
    c, a, r = s["case"], s["a"].float(), s["case"]["rank"]
    masks = [_keep(c["rows"], c["width"], p, s["rng"], s["stream"] + b) for b, p in enumerate(s["p"])]
    x16 = s["x"].to(s["a"].dtype)  # the branch's input under autocast
    x = x16.float()
    if not c["bwd"]:
        u = [scale * (torch.where(keep, x, 0.0) @ a[b * r:(b + 1) * r].T) for b, (keep, scale) in enumerate(masks)]
        return {"x16": x16, "u": torch.cat(u, 1).to(x16.dtype)}
    dx, da = s["addend"], []
    for b, (keep, scale) in enumerate(masks):
        du = s["du"][:, b * r:(b + 1) * r].float()
        dx = dx + torch.where(keep, scale * (du @ a[b * r:(b + 1) * r]), 0.0)
        da.append(scale * (du.T @ torch.where(keep, x, 0.0)))
    return {"dx": dx, "da": torch.cat(da)}


def _tables(s):
    """cos, sin fp32 [tokens, rot] of the case."""
    if s["case"]["op"] == "norm":
        return s["cos"], s["sin"]
    axis = torch.tensor(_axis_of(s["sections"], s["case"]["inter"]), device=s["inv"].device)
    ang = s["positions"][axis].double().T * s["inv"].double()  # far positions: the angle in 64 bits
    cos, sin = ang.cos().float(), ang.sin().float()
    return torch.cat([cos, cos], 1), torch.cat([sin, sin], 1)


def _axis_of(sections, inter):
    """The axis of each frequency: one block after the other, or the axes in turn while they have some left."""
    if not inter:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out, a = list(sections), [], 0
    while len(out) < sum(sections):
        if left[a]:
            left[a] -= 1
            out.append(a)
        a = (a + 1) % len(sections)
    return out


def _rotate(x, cos, sin):
    """x [tokens, heads, dim] fp32, its first cos.shape[1] dims rotated."""
    rot = cos.shape[1]
    y, rest = x[..., :rot], x[..., rot:]
    turned = torch.cat([-y[..., rot // 2:], y[..., :rot // 2]], -1)
    return torch.cat([y * cos[:, None] + turned * sin[:, None], rest], -1)


def _unrotate(g, cos, sin):
    rot = cos.shape[1]
    y, rest = g[..., :rot], g[..., rot:]
    z = y * sin[:, None]
    turned = torch.cat([z[..., rot // 2:], -z[..., :rot // 2]], -1)
    return torch.cat([y * cos[:, None] + turned, rest], -1)


def _plain_rotate(s):
    c = s["case"]
    cos, sin = _tables(s)
    out = {}
    for n, x, w, lora in (("q", s["q"], s["wq"], s["lora"]), ("k", s["k"], s["wk"], None)):
        dt = x.dtype
        x = x.float() if lora is None else x.float() + lora.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) if w is not None else None
        if not c["bwd"]:
            y = x if w is None else x * r * w
            out[n] = _rotate(y, cos, sin).to(dt).transpose(0, 1).contiguous()
            continue
        g = _unrotate(s["g" + n].transpose(0, 1).float(), cos, sin)
        if w is not None:
            out["w" + n] = (g * x * r).sum((0, 1))
            g = g * w
            g = r * (g - x * (r * r) * (g * x).mean(-1, keepdim=True))
        out[n] = g.to(dt)
    return out


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _own(s):
    from decik_b200 import ops

    c = s["case"]
    if c["op"] == "dropout":
        return ops.dropout(s["x"], c["p"], s["rng"], s["stream"], residual=s["residual"])
    if c["op"] == "lora":
        if c["bwd"]:
            dx, da = ops.lora_down_dropout_bwd(s["du"], s["x"], s["a"], s["p"], s["rng"], s["stream"],
                                               addend=s["addend"])
            return {"dx": dx, "da": da}
        x16, u = ops.lora_down_dropout(s["x"], s["a"], s["p"], s["rng"], s["stream"])
        return {"x16": x16, "u": u}
    if c["op"] == "norm":
        if c["bwd"]:
            got = ops.qk_norm_rope_bwd(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"],
                                       s["sin"], q_lora=s["lora"])
        else:
            got = ops.qk_norm_rope_fwd(s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"],
                                       q_lora=s["lora"])
    elif c["bwd"]:
        normed = dict(q=s["q"], k=s["k"], q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"]) if c["norm"] else {}
        got = ops.rope_axes_bwd(s["gq"], s["gk"], s["positions"], s["inv"], s["sections"], interleaved=c["inter"],
                                **normed)
    else:
        got = ops.rope_axes_fwd(s["q"], s["k"], s["positions"], s["inv"], s["sections"], interleaved=c["inter"],
                                q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"])
    return dict(zip(("q", "k", "wq", "wk"), got))


def run(state):
    if own:
        return _own(state)
    return {"dropout": _plain_dropout, "lora": _plain_lora}.get(state["case"]["op"], _plain_rotate)(state)


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_factor(rows, width, p, rng, stream):
    """keep * scale as float64 [rows, width], from unsigned 64-bit integers on the host."""
    seed, off = (int(v) & (2 ** 64 - 1) for v in rng.tolist())
    off = (off + stream) & (2 ** 64 - 1)
    n = rows * width
    u = np.uint64
    m, sh = u(M32), u(32)
    group = np.arange((n + 7) // 8, dtype=u)
    ctr = [group & m, group >> sh, np.full_like(group, off & M32), np.full_like(group, off >> 32)]
    for step in range(7):
        key = [u(((seed & M32) + step * 0x9E3779B9) & M32), u(((seed >> 32) + step * 0xBB67AE85) & M32)]
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> sh) ^ ctr[1] ^ key[0], b & m, (a >> sh) ^ ctr[3] ^ key[1], a & m]
    lanes = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    cut = int(math.floor(p * 65536 + 0.5))
    f = np.where(lanes >= cut, 65536.0 / (65536 - cut), 0.0).reshape(rows, width)
    return torch.from_numpy(f).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("dropout", "lora") and case["rows"] * case["width"] > 60_000_000:
        return None
    if case["op"] == "dropout":
        y = s["x"].double() * _exact_factor(case["rows"], case["width"], case["p"], s["rng"], s["stream"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "lora":
        nb, r = case["branches"], case["rank"]
        f = [_exact_factor(case["rows"], case["width"], s["p"][b], s["rng"], s["stream"] + b) for b in range(nb)]
        a = s["a"].double().view(nb, r, -1)
        x16 = s["x"].to(s["a"].dtype)
        if not case["bwd"]:
            u = torch.stack([torch.einsum("tk,rk->tr", x16.double() * f[b], a[b]) for b in range(nb)], 1)
            return {"x16": x16.double(), "u": u.reshape(case["rows"], nb * r)}
        du = s["du"].double().view(case["rows"], nb, r)
        dx = s["addend"].double() + sum(f[b] * torch.einsum("tr,rk->tk", du[:, b], a[b]) for b in range(nb))
        da = torch.cat([torch.einsum("tr,tk->rk", du[:, b], x16.double() * f[b]) for b in range(nb)])
        return {"dx": dx, "da": da}
    half = case["rot"] // 2
    if case["op"] == "norm":
        c_lo, c_hi = s["cos"].double().split(half, 1)
        s_lo, s_hi = s["sin"].double().split(half, 1)
    else:
        ang = torch.empty(case["tokens"], half, dtype=torch.float64, device="cuda")
        for j, axis in enumerate(_axis_of(s["sections"], case["inter"])):
            ang[:, j] = s["positions"][axis].double() * s["inv"][j].double()
        c_lo = c_hi = ang.cos()
        s_lo = s_hi = ang.sin()
    c_lo, c_hi, s_lo, s_hi = (t[None] for t in (c_lo, c_hi, s_lo, s_hi))
    out = {}
    for n in ("q", "k"):  # head by head first: [heads, tokens, dim]
        x = s[n].transpose(0, 1).double()
        if n == "q" and s["lora"] is not None:
            x = x + s["lora"].transpose(0, 1).double()
        w = s["w" + n].double() if s["w" + n] is not None else None
        rms = (x.pow(2).sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt() if w is not None else None
        if case["bwd"]:
            g = s["g" + n].double()
            lo, hi, rest = g[..., :half], g[..., half:2 * half], g[..., 2 * half:]
            g = torch.cat([lo * c_lo + hi * s_hi, hi * c_hi - lo * s_lo, rest], -1)
            if w is not None:
                xn = x / rms
                out["w" + n] = torch.einsum("htd,htd->d", g, xn)
                g = g * w
                g = (g - xn * (g * xn).mean(-1, keepdim=True)) / rms
            out[n] = g.transpose(0, 1)
        else:
            y = x if w is None else x / rms * w
            lo, hi, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
            out[n] = torch.cat([lo * c_lo - hi * s_lo, hi * c_hi + lo * s_hi, rest], -1)
    return out
