"""The operators of the attention inputs on the GPU against plain 64-bit implementations (oracle/):
counter-based dropout, the LoRA down projections under it, the head norms with the rotation and the
rotation by several axes; forward, backward, strides, empty and long inputs, capture, streams.

Tolerances count roundings. A 16-bit result is off by half a step of its type (eps / 2 relative, or
half the smallest subnormal) plus the fp32 arithmetic before it: a sum of n products is off by at most
about n * 2^-24 of the sum of their magnitudes (2^-23 on the tensor cores, whose additions truncate),
and the few other fp32 operations by 2^-24 each of what they work on."""

import numpy as np
import pytest
import torch

from oracle import dropout as o_drop
from oracle import head_rope as o_rope

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U24, U23 = 2.0 ** -24, 2.0 ** -23
TINY = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}


@pytest.fixture()
def ops(cuda_lib):
    from decik_b200 import ops
    return ops


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(got, want, mag, n, what, unit=U24):
    """|got - want| <= half a step of got's type + n * unit * mag, elementwise."""
    dt = got.dtype
    bound = n * unit * mag + TINY[dt]
    if dt != FP32:
        bound = bound + torch.finfo(dt).eps / 2 * (np.abs(want) + n * unit * mag)
    over = np.abs(_np(got) - want) - bound
    bad = int(np.sum(~(over <= 0)))
    if bad:
        at = np.unravel_index(np.argmax(np.where(np.isnan(over), np.inf, over)), over.shape)
        allowed = float(np.broadcast_to(bound, over.shape)[at])
        pytest.fail(f"{what}: {bad} values off, the worst by {over[at] + allowed:.3e} at {at}, allowed {allowed:.3e}")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rng(seed=3, offset=2 ** 33 + 5):
    return torch.tensor([seed, offset], device="cuda")


# ------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4096, 100003])
@pytest.mark.parametrize("x_dt,res_dt,out_dt", [(BF16, None, None), (FP16, FP32, None), (FP32, None, BF16),
                                                (BF16, BF16, None), (FP32, FP32, None), (FP32, None, None)])
def test_dropout(ops, n, x_dt, res_dt, out_dt):
    g = _gen(n)
    x = torch.randn(n, generator=g, device="cuda").to(x_dt)
    res = None if res_dt is None else torch.randn(n, generator=g, device="cuda").to(res_dt)
    y = ops.dropout(x, 0.3, _rng(), 4, residual=res, out_dtype=out_dt)
    assert y.dtype == (res_dt or out_dt or x_dt)
    want = o_drop.dropout(_np(x), 0.3, 3, 2 ** 33 + 5, 4, None if res is None else _np(res))
    scale = o_drop.cut_scale(0.3)[1]
    # scale, product and sum rounded once each
    _check(y, want, np.abs(_np(x)) * scale + (0 if res is None else np.abs(_np(res))), 3, "dropout")
    if res is None:
        kept = o_drop.keep(n, 0.3, 3, 2 ** 33 + 5, 4)
        assert np.array_equal(_np(y) != 0, kept & (_np(x) != 0))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 0.5, 1.0])
def test_dropout_extreme_p(ops, p):
    x = torch.randn(1000, device="cuda")
    y = ops.dropout(x, p, _rng())
    want = o_drop.dropout(_np(x), p, 3, 2 ** 33 + 5)
    assert np.array_equal(_np(y), want)     # scales 1, 2 and 0: no rounding


def test_dropout_drops_nan_and_inf(ops):
    x = torch.full((64,), float("nan"), device="cuda", dtype=BF16)
    x[::2] = float("inf")
    y = _np(ops.dropout(x, 0.5, _rng()))
    k = o_drop.keep(64, 0.5, 3, 2 ** 33 + 5)
    assert (y[~k] == 0).all() and not np.isfinite(y[k]).any()


@pytest.mark.parametrize("off", [0, 1, 3])
def test_dropout_any_alignment_and_in_place(ops, cuda_lib, off):
    """Buffers that start anywhere; out over x and over the residual."""
    x = torch.randn(1000 + off, device="cuda").to(BF16)[off:]
    r = torch.randn(1000 + 2 * off, device="cuda")[2 * off:]
    want = ops.dropout(x.clone(), 0.2, _rng(), 1, residual=r.clone())
    assert torch.equal(ops.dropout(x, 0.2, _rng(), 1, residual=r), want)
    x32 = x.float()
    s = torch.cuda.current_stream().cuda_stream
    rng = _rng()
    assert cuda_lib.decik_dropout(x.data_ptr(), 1, r.data_ptr(), r.data_ptr(), 2, 1000, 0.2, rng.data_ptr(), 1, s) == 0
    assert torch.equal(r, want)
    w2 = ops.dropout(x32.clone(), 0.2, _rng(), 1)
    assert cuda_lib.decik_dropout(x32.data_ptr(), 2, None, x32.data_ptr(), 2, 1000, 0.2, rng.data_ptr(), 1, s) == 0
    assert torch.equal(x32, w2)


def test_dropout_past_32_bits(ops):
    """Indices above 2^32: the mask's group number and the addresses are 64-bit."""
    n = 2 ** 32 + 8 * 1000 + 3
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.5, _rng(), 2)
    for start in (0, 2 ** 31 - 4000, 2 ** 32 - 4000, n - n % 8 - 4000):
        m = min(8000, n - start)
        k = o_drop.keep(m, 0.5, 3, 2 ** 33 + 5, 2, start=start)
        assert np.array_equal(_np(y[start:start + m]), 2.0 * k)


def test_dropout_empty_and_shapes(ops):
    assert ops.dropout(torch.empty(0, 8, device="cuda"), 0.1, _rng()).shape == (0, 8)
    x = torch.randn(6, 10, 16, device="cuda")
    t = x.transpose(0, 1)                   # row-major order of the view, not of its memory
    assert torch.equal(ops.dropout(t, 0.4, _rng()), ops.dropout(t.contiguous(), 0.4, _rng()))


def test_dropout_refusals_gpu(ops):
    x = torch.randn(8, device="cuda")
    for call in (lambda: ops.dropout(x, 0.1, torch.zeros(2, device="cuda")),
                 lambda: ops.dropout(x, 0.1, torch.zeros(3, dtype=torch.int64, device="cuda")),
                 lambda: ops.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.dropout(x, 1.1, _rng()), lambda: ops.dropout(x.double(), 0.1, _rng()),
                 lambda: ops.dropout(x, 0.1, _rng(), residual=x[:4]),
                 lambda: ops.dropout(x, 0.1, _rng(), residual=x, out_dtype=BF16)):
        with pytest.raises(RuntimeError, match="decik_b200"):
            call()


# ------------------------------------------------------------------------------------ LoRA down projections
LORA = [  # T, W, rank, p of each branch, x dtype, compute dtype
    (1, 64, 16, (0.1, 0.3), FP32, BF16), (7, 8, 8, (0.5,), FP32, FP16), (16, 1536, 16, (0.05, 0.0), FP32, BF16),
    (33, 264, 32, (0.2, 0.6), BF16, BF16), (129, 1000, 64, (0.1,), FP16, FP16), (830, 1536, 16, (0.05, 0.1), FP32, FP16),
    (65, 3584, 24, (0.1, 0.1), FP32, BF16), (1030, 520, 8, (1.0, 0.25), BF16, BF16), (300, 2048, 48, (0.3,), FP32, BF16),
    (2500, 136, 16, (0.1,), FP32, BF16)]


def _lora_case(T, W, rank, p, xd, dt, seed=0):
    g = _gen(seed + T)
    x = torch.randn(T, W, generator=g, device="cuda").to(xd)
    a = (torch.randn(len(p) * rank, W, generator=g, device="cuda") / W ** 0.5).to(dt)
    du = torch.randn(T, len(p) * rank, generator=g, device="cuda").to(dt)
    add = torch.randn(T, W, generator=g, device="cuda")
    return x, a, du, add


@pytest.mark.parametrize("T,W,rank,p,xd,dt", LORA)
def test_lora_down_dropout(ops, T, W, rank, p, xd, dt):
    x, a, _, _ = _lora_case(T, W, rank, p, xd, dt)
    x16, u = ops.lora_down_dropout(x, a, p, _rng(), 6)
    assert torch.equal(x16, x.to(dt)) and u.dtype == dt
    want, mag = o_drop.lora_down(_np(x16), _np(a), p, 3, 2 ** 33 + 5, 6)
    _check(u, want, mag, W + 8, "u", U23)


@pytest.mark.parametrize("with_addend", [False, True])
@pytest.mark.parametrize("T,W,rank,p,xd,dt", LORA)
def test_lora_down_dropout_bwd(ops, T, W, rank, p, xd, dt, with_addend):
    x, a, du, add = _lora_case(T, W, rank, p, xd, dt)
    x16, addend = x.to(dt), add if with_addend else None
    dx, da = ops.lora_down_dropout_bwd(du, x16, a, p, _rng(), 6, addend=addend)
    wdx, wda, mdx, mda = o_drop.lora_down_bwd(_np(du), _np(x16), _np(a), p, 3, 2 ** 33 + 5, 6,
                                              None if addend is None else _np(addend))
    _check(dx, wdx, mdx, rank + 8, "dx", U23)
    _check(da, wda, mda, T + 8, "da", U23)
    dx2, da2 = ops.lora_down_dropout_bwd(du, x16, a, p, _rng(), 6, addend=addend)
    assert torch.equal(dx, dx2) and torch.equal(da, da2)        # fixed order of the sums


def test_lora_long_batch_keeps_its_precision(ops):
    """40,000 tokens. dA is summed in chunks of at most 1,024 tokens on the tensor cores, then 40 chunks in
    fp32, so the count of its roundings stops growing with the batch at 1024 of 2^-23 and 40 of 2^-24 of the
    sum of the magnitudes; a warp of the forward sums W / 8 products, and the 8 warps' sums are added. 8 more
    of each for the scale, as above. The reference runs in 64 bits on the GPU with the mask of ops.dropout."""
    T, W, rank, p = 40000, 3584, 16, (0.1, 0.4)
    x, a, du, add = _lora_case(T, W, rank, p, BF16, BF16)
    dx, da = ops.lora_down_dropout_bwd(du, x, a, p, _rng(), 1, addend=add)
    _, u = ops.lora_down_dropout(x, a, p, _rng(), 1)
    ones = torch.ones(T, W, device="cuda")
    want_dx, mag_dx = add.double(), add.double().abs()
    for b in range(2):
        rows = slice(rank * b, rank * (b + 1))
        keep = ops.dropout(ones, p[b], _rng(), 1 + b).double()
        xm, g, ab = x.double() * keep, du[:, rows].double(), a[rows].double()
        mag = g.abs().T @ xm.abs()
        assert ((da[rows].double() - g.T @ xm).abs() <= (1024 * U23 + 40 * U24 + 8 * U23) * mag).all()
        want, mag = xm @ ab.T, xm.abs() @ ab.abs().T
        bound = (W / 8 + 8 + 8) * U23 * mag
        assert ((u[:, rows].double() - want).abs() <= bound + torch.finfo(BF16).eps / 2 * (want.abs() + bound)).all()
        want_dx += keep * (g @ ab)
        mag_dx += keep * (g.abs() @ ab.abs())
    assert ((dx.double() - want_dx).abs() <= (2 * rank + 8) * U23 * mag_dx).all()


def test_lora_gradients_are_the_forwards_differences(ops):
    """dA and dx against differences of the forward's u (fp32 differences of a 16-bit u: a linear
    function, so a large step is exact up to u's roundings)."""
    T, W, rank, p = 24, 64, 8, (0.25, 0.5)
    x, a, du, _ = _lora_case(T, W, rank, p, FP16, FP16)
    dx, da = ops.lora_down_dropout_bwd(du, x, a, p, _rng(), 0)
    loss = lambda x, a: (ops.lora_down_dropout(x, a, p, _rng(), 0)[1].double() * du.double()).sum().item()
    base_mag = (ops.lora_down_dropout(x, a, p, _rng(), 0)[1].double() * du.double()).abs().sum().item()
    for t, k, r in [(0, 0, 0), (5, 9, 3), (23, 63, 15), (11, 32, 8)]:
        for ten, i, grad in ((x, (t, k), dx), (a, (r, k), da)):
            up, h = ten.clone(), 64.0
            up[i] += h
            step = (up[i] - ten[i]).item()
            got = (loss(up, a) if ten is x else loss(x, up)) - loss(x, a)
            # each u is rounded once on both sides: half a step of fp16 relative to |u|, at most |u| + |change|
            slack = 2.0 ** -11 * (2 * base_mag + abs(got) * 2) + 2.0 ** -11 * abs(step) * du.abs().max().item() * 64
            assert abs(got - step * grad[i].item()) <= slack


def test_lora_strides_and_in_place_addend(ops):
    T, W, rank, p = 70, 128, 16, (0.1, 0.2)
    x, a, du, add = _lora_case(T, W, rank, p, BF16, BF16)
    wide = torch.zeros(T, W + 64, dtype=BF16, device="cuda")
    wide[:, 32:32 + W] = x
    wa = torch.zeros(2 * rank, W + 8, dtype=BF16, device="cuda")
    wa[:, 8:] = a
    wdu = torch.zeros(T, 96, dtype=BF16, device="cuda")
    wdu[:, 64:] = du
    _, u = ops.lora_down_dropout(x, a, p, _rng())
    assert torch.equal(ops.lora_down_dropout(wide[:, 32:32 + W], wa[:, 8:], p, _rng())[1], u)
    dx, da = ops.lora_down_dropout_bwd(du, x, a, p, _rng(), addend=add)
    buf = torch.zeros(T + 1, W + 4, device="cuda")
    buf[:T, 4:] = add
    dx2, da2 = ops.lora_down_dropout_bwd(wdu[:, 64:], wide[:, 32:32 + W], wa[:, 8:], p, _rng(), addend=buf[:T, 4:],
                                         out=buf[:T, 4:])
    assert torch.equal(dx2, dx) and torch.equal(da2, da)
    assert not buf[T].any() and not buf[:, :4].any()            # nothing written around the rows


def test_lora_masked_values_do_not_reach_the_results(ops):
    """NaN in an input that a branch drops leaves that branch's u alone."""
    T, W = 4, 64
    x, a, du, _ = _lora_case(T, W, 16, (0.5, 0.5), BF16, BF16)
    kept = [o_drop.keep(T * W, 0.5, 3, 2 ** 33 + 5, b).reshape(T, W) for b in (0, 1)]
    t, k = np.argwhere(~kept[0] & kept[1])[0]
    bad = x.clone()
    bad[t, k] = float("nan")
    _, u0 = ops.lora_down_dropout(x, a, (0.5, 0.5), _rng())
    _, u1 = ops.lora_down_dropout(bad, a, (0.5, 0.5), _rng())
    assert torch.equal(u1[:, :16], u0[:, :16]) and torch.isnan(u1[t, 16:]).all()
    rest = [i for i in range(T) if i != t]
    assert torch.equal(u1[rest], u0[rest])
    da = ops.lora_down_dropout_bwd(du, bad, a, (0.5, 0.5), _rng())[1]
    assert not torch.isnan(da[:16]).any() and torch.isnan(da[16:, k]).all()


def test_lora_empty(ops):
    a = torch.randn(32, 64, device="cuda").to(BF16)
    x = torch.empty(0, 64, device="cuda")
    x16, u = ops.lora_down_dropout(x, a, (0.1, 0.1), _rng())
    assert x16.shape == (0, 64) and u.shape == (0, 32)
    dx, da = ops.lora_down_dropout_bwd(u, x16, a, (0.1, 0.1), _rng())
    assert dx.shape == (0, 64) and not da.any()


def test_lora_refusals_gpu(ops):
    x, a, du, add = _lora_case(8, 64, 16, (0.1, 0.1), FP32, BF16)
    p, x16 = (0.1, 0.1), x.to(BF16)
    for call in (lambda: ops.lora_down_dropout(x.double(), a, p, _rng()), lambda: ops.lora_down_dropout(x[0], a, p, _rng()),
                 lambda: ops.lora_down_dropout(x[:, :32], a, p, _rng()),
                 lambda: ops.lora_down_dropout(x, a, (0.1, 0.1, 0.1), _rng()),
                 lambda: ops.lora_down_dropout(x, a.float(), p, _rng()),
                 lambda: ops.lora_down_dropout(x[:, 1:61], a[:, 1:61], p, _rng()),
                 lambda: ops.lora_down_dropout(x, a, p, _rng().cpu()),
                 lambda: ops.lora_down_dropout(x[:1].expand(8, 64), a, p, _rng()),
                 lambda: ops.lora_down_dropout_bwd(du[:4], x16, a, p, _rng()),
                 lambda: ops.lora_down_dropout_bwd(du, x, a, p, _rng()),
                 lambda: ops.lora_down_dropout_bwd(du, x16, a, p, _rng(), addend=add[:4]),
                 lambda: ops.lora_down_dropout_bwd(du, x16, a, p, _rng(), out=add.to(BF16))):
        with pytest.raises(RuntimeError, match="decik_b200"):
            call()


# ------------------------------------------------------------------------------------ head norms and rotation
HEADS = [  # T, Hq, Hk, D, R, dtype
    (1, 12, 2, 128, 128, BF16), (5, 1, 1, 16, 16, FP16), (37, 3, 1, 32, 16, BF16), (130, 8, 2, 64, 64, FP16),
    (33, 14, 2, 80, 48, BF16), (77, 6, 3, 96, 96, FP16), (19, 4, 4, 256, 128, BF16), (830, 12, 2, 128, 128, FP16),
    (4097, 5, 1, 112, 64, BF16)]


def _heads_case(T, Hq, Hk, D, R, dt, seed=0, lora=False):
    g = _gen(seed + T + D)
    proj = (torch.randn(T, Hq + 2 * Hk, D, generator=g, device="cuda") * 1.5
            + torch.randn(D, generator=g, device="cuda")).to(dt)
    s = dict(q=proj[:, :Hq], k=proj[:, Hq:Hq + Hk], eps=1e-6,
             wq=1 + 0.3 * torch.randn(D, generator=g, device="cuda"),
             wk=1 + 0.3 * torch.randn(D, generator=g, device="cuda"),
             ql=(0.2 * torch.randn(T, Hq, D, generator=g, device="cuda")).to(dt) if lora else None,
             gq=torch.randn(Hq, T, D, generator=g, device="cuda").to(dt),
             gk=torch.randn(Hk, T, D, generator=g, device="cuda").to(dt))
    ang = torch.rand(T, R, generator=g, device="cuda") * 6.3
    return dict(s, cos=ang.cos(), sin=ang.sin())


def _x(s, n):
    x = _np(s[n])
    return x + _np(s["ql"]) if n == "q" and s["ql"] is not None else x


def _check_fwd(got, s, cos, sin, normed=True):
    for n, y in zip("qk", got):
        want, mag = o_rope.forward(_x(s, n), _np(s["w" + n]) if normed else None, s["eps"], cos, sin)
        # the mean of D squares, rsqrt, two products, the angle's two roundings, the rotation
        _check(y.transpose(0, 1), want, mag, s["q"].shape[2] + 32, n)


def _check_bwd(got, s, cos, sin, normed=True):
    T, _, D = s["q"].shape
    for n, d in zip("qk", got):
        w = _np(s["w" + n]) if normed else None
        want, mag, dw, mdw = o_rope.backward(_np(s["g" + n].transpose(0, 1)), _x(s, n), w, s["eps"], cos, sin)
        _check(d, want, mag, 2 * D + 48, "d" + n)
        if normed:
            _check(got[2 if n == "q" else 3], dw, mdw, T * s[n].shape[1] + D + 32, "dw" + n)


@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,dt", HEADS)
def test_qk_norm_rope(ops, T, Hq, Hk, D, R, dt, lora):
    s = _heads_case(T, Hq, Hk, D, R, dt, lora=lora)
    cos, sin = _np(s["cos"]), _np(s["sin"])
    args = (s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"])
    _check_fwd(ops.qk_norm_rope_fwd(*args, q_lora=s["ql"]), s, cos, sin)
    got = ops.qk_norm_rope_bwd(s["gq"], s["gk"], *args, q_lora=s["ql"])
    _check_bwd(got, s, cos, sin)
    again = ops.qk_norm_rope_bwd(s["gq"], s["gk"], *args, q_lora=s["ql"])
    assert all(torch.equal(a, b) for a, b in zip(got, again))   # fixed order of the sums


@pytest.mark.parametrize("w_dt", [BF16, FP16])
def test_qk_norm_rope_weight_types(ops, w_dt):
    s = _heads_case(40, 4, 2, 64, 64, BF16)
    s["wq"], s["wk"] = s["wq"].to(w_dt), s["wk"].to(w_dt)
    args = (s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"])
    cos, sin = _np(s["cos"]), _np(s["sin"])
    _check_fwd(ops.qk_norm_rope_fwd(*args), s, cos, sin)
    _check_bwd(ops.qk_norm_rope_bwd(s["gq"], s["gk"], *args), s, cos, sin)


def test_qk_norm_rope_agrees_with_rope(ops):
    """With weights of the rows' own norm the norm does nothing: the rotation is rope_fwd's to its roundings."""
    T, Hq, Hk, D = 50, 4, 2, 128
    s = _heads_case(T, Hq, Hk, D, D, BF16)
    s["q"] = torch.where(torch.randn(T, Hq, D, device="cuda") > 0, 1.0, -1.0).to(BF16)  # mean square 1
    s["k"] = torch.where(torch.randn(T, Hk, D, device="cuda") > 0, 1.0, -1.0).to(BF16)
    one = torch.ones(D, device="cuda")
    got = ops.qk_norm_rope_fwd(s["q"], s["k"], one, one, 0.0, s["cos"], s["sin"])
    want = ops.rope_fwd(s["q"].reshape(T, -1), None, s["k"].reshape(T, -1), s["cos"], s["sin"], Hq, Hk)
    for a, b in zip(got, want):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -7     # one bf16 step of values up to 2


@pytest.mark.parametrize("T,Hq,Hk,D,dt,lora", [(8003, 12, 2, 128, BF16, False), (8003, 16, 4, 64, FP16, False),
                                               (3001, 8, 3, 256, BF16, True), (600, 12, 2, 128, BF16, False)])
def test_norm_weight_gradients_lose_no_part(ops, T, Hq, Hk, D, dt, lora):
    """The weights' gradients of a batch that fills the GPU, with terms of one sign, so that a partial sum that
    is lost or counted twice shows. Roundings: a warp's rows of one part in a chain (at most its share of all
    rows), the CTA's lanes that hold the same values, the CTAs in 64 chains and a tree of 6; each term has
    those of r (the mean of D squares) and a few products."""
    s = _heads_case(T, Hq, Hk, D, D, dt, lora=lora)
    s["cos"], s["sin"] = torch.ones(T, D, device="cuda"), torch.zeros(T, D, device="cuda")
    for n in "qk":
        x = s[n].float() + (s["ql"].float() if n == "q" and lora else 0.0)
        s["g" + n] = (s["g" + n].float().abs() * torch.sign(x).transpose(0, 1)).to(dt).contiguous()
    got = ops.qk_norm_rope_bwd(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"],
                               q_lora=s["ql"])
    lanes = 4 if D <= 64 else 8 if D <= 128 else 16
    ctas = torch.cuda.get_device_properties(0).multi_processor_count * (3 if lora else 4)
    rows = -(-T * lanes // 32) * (Hq + Hk)
    chain = -(-rows // (4 * ctas)) + 128 // lanes + -(-ctas // 64) + 6
    for n, dw in zip("qk", got[2:]):
        g, x = s["g" + n].transpose(0, 1).double(), torch.as_tensor(_x(s, n), device="cuda")
        want = (g * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])).sum((0, 1)).cpu().numpy()
        assert (want > 0).all()
        _check(dw, want, want, chain + D + 32, "dw" + n)


def test_qk_norm_rope_views(ops):
    """Head-major and padded inputs, broadcast gradients, one row."""
    s = _heads_case(33, 4, 2, 64, 32, BF16)
    tail = (s["wq"], s["wk"], s["eps"], s["cos"], s["sin"])
    want = ops.qk_norm_rope_fwd(s["q"], s["k"], *tail)
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    pad = torch.zeros(33, 7, 72, dtype=BF16, device="cuda")
    pad[:, 1:5, :64] = s["q"]
    for q in (hm(s["q"]), pad[:, 1:5, :64]):
        got = ops.qk_norm_rope_fwd(q, hm(s["k"]), *tail)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    g1 = torch.randn(1, 33, 64, device="cuda").to(BF16)
    wide = ops.qk_norm_rope_bwd(g1.expand(4, 33, 64), g1.expand(2, 33, 64), s["q"], s["k"], *tail)
    full = ops.qk_norm_rope_bwd(g1.repeat(4, 1, 1), g1.repeat(2, 1, 1), s["q"], s["k"], *tail)
    assert all(torch.equal(a, b) for a, b in zip(wide, full))
    one = s["q"][:1].as_strided((1, 4, 64), (1, s["q"].stride(1), 1))   # a stride nobody reads
    got = ops.qk_norm_rope_fwd(one, s["k"][:1], s["wq"], s["wk"], s["eps"], s["cos"][:1], s["sin"][:1])
    assert torch.equal(got[0], want[0][:, :1])


def test_qk_norm_rope_extreme_rows(ops):
    """A row of zeros (eps alone under the root), one of the largest values, one with a NaN: the others
    stay as they are."""
    s = _heads_case(8, 2, 1, 64, 64, BF16)
    args = lambda q: (q, s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"])
    base = ops.qk_norm_rope_fwd(*args(s["q"]))[0]
    q = s["q"].contiguous().clone()
    q[1, 0], q[3, 1], q[5, 0, 7] = 0.0, 2.0 ** 60, float("nan")
    got = ops.qk_norm_rope_fwd(*args(q))[0]
    assert not got[0, 1].any() and torch.isnan(got[0, 5]).all() and torch.isfinite(got[1, 3]).all()
    for h, t in [(h, t) for h in range(2) for t in range(8) if (t, h) not in ((1, 0), (3, 1), (5, 0))]:
        assert torch.equal(got[h, t], base[h, t])
    dq = ops.qk_norm_rope_bwd(s["gq"], s["gk"], *args(torch.zeros_like(q)))[0]
    assert torch.isfinite(dq.float()).all()


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("sections_n,inter,far,pos_dt", [(1, False, 100, torch.int64), (3, False, 5000, torch.int32),
                                                         (3, True, 2 ** 20, torch.int64), (4, True, 2 ** 30, torch.int32),
                                                         (2, False, 2 ** 40, torch.int64)])
@pytest.mark.parametrize("T,Hq,Hk,D,R,dt", [HEADS[0], HEADS[3], HEADS[4], HEADS[6], HEADS[8]])
def test_rope_axes(ops, T, Hq, Hk, D, R, dt, sections_n, inter, far, pos_dt, normed):
    s = _heads_case(T, Hq, Hk, D, R, dt, lora=normed)
    part = (R // 2) // (sections_n + 1)
    sections = (R // 2 - part * (sections_n - 1),) + (part,) * (sections_n - 1)
    g = _gen(9)
    pos = torch.randint(-far if pos_dt == torch.int64 else 0, far, (sections_n, T), generator=g, device="cuda").to(pos_dt)
    inv = (1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)).float()
    cos, sin = o_rope.axes_cos_sin(pos.cpu().numpy(), _np(inv), sections, inter)
    norm = dict(q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"]) if normed else {}
    got = ops.rope_axes_fwd(s["q"], s["k"], pos, inv, sections, inter, q_lora=s["ql"], **norm)
    bwd = ops.rope_axes_bwd(s["gq"], s["gk"], pos, inv, sections, inter, q_lora=s["ql"],
                            **(dict(norm, q=s["q"], k=s["k"]) if normed else {}))
    assert len(bwd) == (4 if normed else 2)
    if far <= 2 ** 32:
        _check_fwd(got, s, cos, sin, normed)
        _check_bwd(bwd, s, cos, sin, normed)
        return
    # position * inv_freq is rounded to 2^-53 of up to 2^40 on both sides, which moves the angle by up to
    # 2 * 2^-13; out = y cos - z sin moves by at most that times |y sin| + |z cos| <= |y| + |z|
    ones = np.ones_like(cos)
    for n, y in zip("qk", got):
        w = _np(s["wq" if n == "q" else "wk"]) if normed else None
        want, _ = o_rope.forward(_x(s, n), w, s["eps"], cos, sin)
        _, both = o_rope.forward(_x(s, n), w, s["eps"], ones, ones)
        _check(y.transpose(0, 1), want, both, 2.0 ** -12 / U24 + D + 32, n)


def test_rope_axes_one_axis_is_rope(ops):
    """Positions of one axis against the tables: rope_fwd's result to one 16-bit step."""
    s = _heads_case(100, 4, 2, 128, 128, BF16)
    inv = (1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device="cuda") / 128)).float()
    pos = torch.arange(100, device="cuda")
    ang = torch.cat([pos[:, None].double() * inv.double()] * 2, 1)
    got = ops.rope_axes_fwd(s["q"], s["k"], pos, inv, (64,))
    want = ops.rope_fwd(s["q"].reshape(100, -1).contiguous(), None, s["k"].reshape(100, -1).contiguous(),
                        ang.cos().float(), ang.sin().float(), 4, 2)
    for a, b in zip(got, want):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * b.float().abs().max()


def test_rope_axes_position_views(ops):
    s = _heads_case(64, 2, 1, 64, 64, FP16)
    inv = torch.rand(32, device="cuda")
    pos = torch.randint(0, 999, (3, 64), device="cuda")
    want = ops.rope_axes_fwd(s["q"], s["k"], pos, inv, (16, 8, 8))
    wide = torch.zeros(3, 100, dtype=torch.int64, device="cuda")
    wide[:, 20:84] = pos
    for p in (wide[:, 20:84], pos.t().contiguous().t(), pos.to(torch.int32)):
        assert all(torch.equal(a, b) for a, b in zip(ops.rope_axes_fwd(s["q"], s["k"], p, inv, (16, 8, 8)), want))
    same = pos[:1].expand(3, 64)    # one row of positions for all axes
    a = ops.rope_axes_fwd(s["q"], s["k"], same, inv, (16, 8, 8))
    b = ops.rope_axes_fwd(s["q"], s["k"], pos[0], inv, (32,))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


BEHIND = [(80, 48, BF16), (64, 32, FP16), (256, 16, BF16), (112, 96, FP16)]   # D, R, dtype


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("D,R,dt", BEHIND)
def test_values_behind_the_rotated_ones_stay_apart(ops, D, R, dt, lora, bad):
    """An infinity or NaN behind rotary_dim comes out at its own place, and every other value of the row, and
    of the gradient through the plain rotation, keeps its bits."""
    T, H = 21, 2
    s = _heads_case(T, H, 1, D, R, dt, lora=lora)
    pos, inv = torch.randint(0, 999, (2, T), generator=_gen(4), device="cuda"), torch.rand(R // 2, device="cuda")
    sections = (R // 2 - 3, 3)
    for d in sorted({R, R + 3, R + 8, D - 9, D - 1}):
        if d < R:
            continue
        q, gq = s["q"].clone(), s["gq"].clone()
        q[5, 1, d] = gq[1, 5, d] = bad
        fwd = lambda q: ops.rope_axes_fwd(q, s["k"], pos, inv, sections, q_lora=s["ql"])
        bwd = lambda g: ops.rope_axes_bwd(g, s["gk"], pos, inv, sections)
        for got, want in ((fwd(q)[0].transpose(0, 1), fwd(s["q"])[0].transpose(0, 1)), (bwd(gq)[0], bwd(s["gq"])[0])):
            assert torch.equal(torch.nan_to_num(got[5, 1, d], nan=7.0), torch.nan_to_num(torch.tensor(
                bad, dtype=dt, device="cuda"), nan=7.0))
            got[5, 1, d] = want[5, 1, d]
            assert torch.equal(got, want), d


@pytest.mark.parametrize("axes", [False, True])
@pytest.mark.parametrize("D,R,dt", BEHIND)
def test_normed_values_behind_the_rotated_ones_stay_apart(ops, D, R, dt, axes):
    """The same with norms: a weight's NaN reaches its own place of each row alone, an infinity of x makes the
    row's other values 0 (the mean is infinite), a gradient's infinity leaves the sums of the other
    weights' gradients as they were."""
    T, H = 40, 3
    s = _heads_case(T, H, 1, D, R, dt)
    pos, inv = torch.randint(0, 999, (2, T), generator=_gen(4), device="cuda"), torch.rand(R // 2, device="cuda")
    sections, inf = (R // 2 - 3, 3), float("inf")
    for d in sorted({R, R + 3, R + 8, D - 9, D - 1}):
        if d < R:
            continue

        def fwd(q, wq):
            if axes:
                return ops.rope_axes_fwd(q, s["k"], pos, inv, sections, q_weight=wq, k_weight=s["wk"], eps=1e-6)[0]
            return ops.qk_norm_rope_fwd(q, s["k"], wq, s["wk"], 1e-6, s["cos"], s["sin"])[0]

        def dwq(gq):
            if axes:
                return ops.rope_axes_bwd(gq, s["gk"], pos, inv, sections, q=s["q"], k=s["k"], q_weight=s["wq"],
                                         k_weight=s["wk"], eps=1e-6)[2]
            return ops.qk_norm_rope_bwd(gq, s["gk"], s["q"], s["k"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])[2]

        rest = [i for i in range(D) if i != d]
        want, w = fwd(s["q"], s["wq"]), s["wq"].clone()
        w[d] = float("nan")
        got = fwd(s["q"], w)
        assert torch.isnan(got[..., d]).all() and torch.equal(got[..., rest], want[..., rest])
        q = s["q"].clone()
        q[5, 1, d] = inf
        got = fwd(q, s["wq"])
        assert torch.isnan(got[1, 5, d]) and not got[1, 5, rest].any()
        got[1, 5] = want[1, 5]
        assert torch.equal(got, want)
        want, gq = dwq(s["gq"]), s["gq"].clone()
        gq[1, 5, d] = inf
        got = dwq(gq)
        assert not torch.isfinite(got[d]) and torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_rope_axes_inv_freq_slices(ops, off, normed):
    """inv_freq as a slice of a longer table, wherever it starts: the same bits."""
    s = _heads_case(40, 4, 2, 64, 64, BF16)
    table = torch.rand(40, generator=_gen(3), device="cuda")
    pos = torch.randint(0, 999, (3, 40), generator=_gen(4), device="cuda")
    part = table[off:off + 32]
    assert part.data_ptr() % 16 == 4 * off
    norm = dict(q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"]) if normed else {}
    saved = dict(norm, q=s["q"], k=s["k"]) if normed else {}
    run = lambda inv: (ops.rope_axes_fwd(s["q"], s["k"], pos, inv, (16, 8, 8), **norm)
                       + ops.rope_axes_bwd(s["gq"], s["gk"], pos, inv, (16, 8, 8), **saved))
    for a, b in zip(run(part), run(part.clone())):
        assert torch.equal(a, b)


def test_heads_empty(ops):
    s = _heads_case(4, 2, 1, 64, 64, BF16)
    args = (s["q"][:0], s["k"][:0], s["wq"], s["wk"], s["eps"], s["cos"][:0], s["sin"][:0])
    q, k = ops.qk_norm_rope_fwd(*args)
    assert q.shape == (2, 0, 64) and k.shape == (1, 0, 64)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(q, k, *args)
    assert dq.shape == (0, 2, 64) and not dwq.any() and not dwk.any()
    pos = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    assert ops.rope_axes_fwd(s["q"][:0], s["k"][:0], pos, torch.ones(32, device="cuda"), (32,))[0].shape == (2, 0, 64)


def test_heads_past_32_bits(ops):
    """More than 2^31 values in the queries: the last tokens."""
    T, Hq, Hk, D = 72000, 120, 8, 256
    g = _gen(0)
    q = torch.randn(T, Hq, D, generator=g, device="cuda", dtype=BF16)
    k = torch.randn(T, Hk, D, generator=g, device="cuda", dtype=BF16)
    w = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    pos = torch.arange(T, device="cuda")[None]
    inv = torch.rand(D // 2, generator=g, device="cuda")
    oq, ok = ops.rope_axes_fwd(q, k, pos, inv, (D // 2,), q_weight=w, k_weight=w, eps=1e-6)
    n = 3
    cos, sin = o_rope.axes_cos_sin(pos[:, -n:].cpu().numpy(), _np(inv), (D // 2,))
    want, mag = o_rope.forward(_np(q[-n:]), _np(w), 1e-6, cos, sin)
    _check(oq[:, -n:].transpose(0, 1), want, mag, D + 32, "q")
    del q, k, ok
    gq = oq
    dq, dk = ops.rope_axes_bwd(gq, gq[:Hk], pos, inv, (D // 2,))
    want, mag, _, _ = o_rope.backward(_np(gq[:, -n:].transpose(0, 1)), None, None, 0.0, cos, sin)
    _check(dq[-n:], want, mag, D + 32, "dq")


def test_heads_refusals_gpu(ops):
    s = _heads_case(8, 2, 1, 64, 64, BF16)
    inv, pos = torch.ones(32, device="cuda"), torch.zeros(3, 8, dtype=torch.int64, device="cuda")
    nf = lambda **o: ops.qk_norm_rope_fwd(**dict(dict(q=s["q"], k=s["k"], q_weight=s["wq"], k_weight=s["wk"], eps=1e-6,
                                                      cos=s["cos"], sin=s["sin"]), **o))
    ax = lambda **o: ops.rope_axes_fwd(**dict(dict(q=s["q"], k=s["k"], positions=pos, inv_freq=inv,
                                                   sections=(16, 8, 8)), **o))
    odd = torch.zeros(8, 2, 65, dtype=BF16, device="cuda")[:, :, 1:]
    for call in (lambda: nf(q=s["q"].float()), lambda: nf(k=s["k"][:4]), lambda: nf(q=odd), lambda: nf(q=s["q"][:, :, ::2]),
                 lambda: nf(q_lora=s["k"]), lambda: nf(q_weight=s["wq"][:32]), lambda: nf(k_weight=s["wk"].to(BF16)),
                 lambda: nf(cos=s["cos"][:4]), lambda: nf(sin=s["sin"].to(BF16)), lambda: nf(eps=-1.0),
                 lambda: nf(q_weight=s["wq"].cpu()), lambda: ax(sections=(16, 8)), lambda: ax(sections=(16, 8, 9)),
                 lambda: ax(positions=pos.float()), lambda: ax(positions=pos[:, :4]), lambda: ax(inv_freq=inv[:16]),
                 lambda: ax(inv_freq=inv.double()), lambda: ax(q_weight=s["wq"]), lambda: ax(positions=pos.cpu()),
                 lambda: ops.rope_axes_bwd(s["gq"], s["gk"], pos, inv, (16, 8, 8), q_weight=s["wq"], k_weight=s["wk"]),
                 lambda: ops.rope_axes_bwd(s["gq"], s["gk"][:, :4], pos, inv, (16, 8, 8)),
                 lambda: ops.qk_norm_rope_bwd(s["gq"].float(), s["gk"], s["q"], s["k"], s["wq"], s["wk"], 1e-6, s["cos"],
                                              s["sin"])):
        with pytest.raises(RuntimeError, match="decik_b200"):
            call()


# ------------------------------------------------------------------------------------ together, as they are used
def _chain(x, a_q, a_v, b_q, w_q, w_k, wq, wk, rng, pos, inv, sections, heads, kv):
    """LoRA'd projection under dropout -> norms and rotation -> packed attention -> residual dropout, as a
    layer of the framework's kind runs them."""
    from decik_b200.solution.attn import AxesRope
    from decik_b200.solution.dropout import CounterDropout, LoRADownDropout
    from decik_b200.solution.varlen import VarlenSDPA

    T = x.shape[0]
    u = LoRADownDropout.apply(x, (0.1, 0.2), rng, 0, BF16, a_q, a_v)
    x16 = x.to(BF16)
    q = torch.nn.functional.linear(x16, w_q).view(T, heads, -1)
    ql = torch.nn.functional.linear(u[:, :16], b_q).view(T, heads, -1)
    k = torch.nn.functional.linear(x16, w_k).view(T, kv, -1)
    q, k = AxesRope.apply(q, ql, k, pos, inv, sections, True, wq, wk, 1e-6)
    cu = torch.tensor([0, T // 3, T], dtype=torch.int32, device=x.device)
    o = VarlenSDPA.apply(q, k, k, cu, T - T // 3, heads // kv, None)
    return CounterDropout.apply(o.reshape(T, -1).float(), 0.1, rng, 2, x), u


def _chain_inputs(T=200, W=512, heads=4, kv=2, D=128):
    g = _gen(11)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    leaf = lambda t: t.requires_grad_(True)
    x = leaf(rn(T, W))
    pos = torch.randint(0, 300, (3, T), generator=g, device="cuda")
    inv = (1e4 ** (-torch.arange(0, D, 2, device="cuda") / D))
    return dict(x=x, a_q=leaf(rn(16, W) / W ** 0.5), a_v=leaf(rn(16, W) / W ** 0.5), b_q=(rn(heads * D, 16) * 0.1).to(BF16),
                w_q=(rn(heads * D, W) / W ** 0.5).to(BF16), w_k=(rn(kv * D, W) / W ** 0.5).to(BF16),
                wq=leaf(1 + 0.1 * rn(D)), wk=leaf(1 + 0.1 * rn(D)), pos=pos, inv=inv, sections=(32, 16, 16), heads=heads,
                kv=kv)


def test_chain_runs_and_its_gradients_are_deterministic_in_the_state(ops):
    from decik_b200.solution.dropout import CounterRNG

    c = _chain_inputs()
    leaves = [c[n] for n in ("x", "a_q", "a_v", "wq", "wk")]

    def step(state):
        y, u = _chain(rng=state, **c)
        return y.detach(), torch.autograd.grad((y * y).sum() + u.float().sum(), leaves)

    r = CounterRNG(5)
    s0, s1 = r.take(3), r.take(3)
    assert s0.tolist() == [5, 0] and s1.tolist() == [5, 3]
    y0, g0 = step(s0)
    y1, g1 = step(s0.clone())
    y2, _ = step(s1)
    assert torch.equal(y0, y1) and not torch.equal(y0, y2)
    assert all(torch.isfinite(t).all() and t.any() for t in g0)
    for a, b in zip(g0, g1):    # the attention backward's fp32 reductions have no fixed order
        assert (a - b).norm() <= 1e-2 * a.norm()


def test_autograd_functions_match_the_oracle(ops):
    """The Functions' gradients, each alone, against the 64-bit formulas."""
    from decik_b200.solution.attn import AxesRope, QKNormRope
    from decik_b200.solution.dropout import CounterDropout, LoRADownDropout

    s = _heads_case(60, 4, 2, 64, 64, BF16, lora=True)
    ins = [s[n].detach().clone().requires_grad_(True) for n in ("q", "ql", "k", "wq", "wk")]
    q, k = QKNormRope.apply(*ins, s["eps"], s["cos"], s["sin"])
    assert q.shape == (1, 4, 60, 64)
    torch.autograd.backward([q, k], [s["gq"][None], s["gk"][None]])
    _check_bwd([ins[0].grad, ins[2].grad, ins[3].grad, ins[4].grad], s, _np(s["cos"]), _np(s["sin"]))
    assert torch.equal(ins[1].grad, ins[0].grad)
    ins = [s[n].detach().clone().requires_grad_(True) for n in ("q", "k")]
    inv, pos = torch.rand(32, device="cuda"), torch.randint(0, 500, (2, 60), device="cuda")
    q, k = AxesRope.apply(ins[0], None, ins[1], pos, inv, (20, 12))
    torch.autograd.backward([q, k], [s["gq"][None], s["gk"][None]])
    cos, sin = o_rope.axes_cos_sin(pos.cpu().numpy(), _np(inv), (20, 12))
    _check_bwd([t.grad for t in ins], dict(s, ql=None), cos, sin, normed=False)
    x, res = torch.randn(50, 24, device="cuda", dtype=BF16).requires_grad_(True), torch.randn(50, 24, device="cuda").requires_grad_(True)
    g = torch.randn(50, 24, device="cuda")
    CounterDropout.apply(x, 0.4, _rng(), 7, res).backward(g)
    assert torch.equal(res.grad, g)
    _check(x.grad, o_drop.dropout(_np(g), 0.4, 3, 2 ** 33 + 5, 7), np.abs(_np(g)) * 2, 3, "dx")
    x = torch.randn(40, 64, device="cuda").requires_grad_(True)
    a = [torch.randn(16, 64, device="cuda").requires_grad_(True) for _ in range(2)]
    du = torch.randn(40, 32, device="cuda").to(BF16)
    LoRADownDropout.apply(x, (0.3, 0.1), _rng(), 1, BF16, *a).backward(du)
    wdx, wda, mdx, mda = o_drop.lora_down_bwd(_np(du), _np(x.to(BF16)), _np(torch.cat(a).to(BF16)), (0.3, 0.1), 3,
                                              2 ** 33 + 5, 1)
    _check(x.grad, wdx, mdx, 24, "dx", U23)
    _check(torch.cat([w.grad for w in a]), wda, mda, 48, "da", U23)


@pytest.mark.parametrize("p", [0.3, (0.3, 0.3), [0.3, 0.3]], ids=["number", "tuple", "list"])
def test_lora_down_dropout_function_gives_each_weight_its_mask(ops, p):
    """One p for two weights: two branches with masks of their own, as in the oracle, both ways."""
    from decik_b200.solution.dropout import LoRADownDropout

    x, a, du, _ = _lora_case(40, 64, 24, (0.3, 0.3), FP32, BF16)
    x.requires_grad_(True)
    ws = [w.float().requires_grad_(True) for w in a.split(24)]
    u = LoRADownDropout.apply(x, p, _rng(), 1, BF16, *ws)
    u.backward(du)
    x16 = _np(x.to(BF16))
    want, mag = o_drop.lora_down(x16, _np(a), (0.3, 0.3), 3, 2 ** 33 + 5, 1)
    _check(u, want, mag, 64 + 8, "u", U23)
    wdx, wda, mdx, mda = o_drop.lora_down_bwd(_np(du), x16, _np(a), (0.3, 0.3), 3, 2 ** 33 + 5, 1)
    _check(x.grad, wdx, mdx, 24 + 8, "dx", U23)
    _check(torch.cat([w.grad for w in ws]), wda, mda, 40 + 8, "da", U23)


def test_functions_take_tensors_off_16_bytes(ops):
    """Inputs and gradients that are contiguous but start off a 16-byte boundary (the slices that a cat's
    backward hands out), and rows of other strides: the aligned tensors' results."""
    from decik_b200.solution.attn import AxesRope, QKNormRope
    from decik_b200.solution.dropout import LoRADownDropout

    def off(t):
        b = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")[3:].view(t.shape)
        assert b.data_ptr() % 16 != 0
        return b.copy_(t)

    s = _heads_case(20, 4, 2, 64, 64, BF16, lora=True)
    inv, pos = torch.rand(32, device="cuda"), torch.randint(0, 500, (2, 20), device="cuda")
    x, a, du, _ = _lora_case(20, 128, 16, (0.3, 0.1), BF16, BF16)
    first = torch.zeros(3, dtype=BF16, device="cuda")
    seen = []

    def run(place, join):
        q, ql, k = (place(s[n]).requires_grad_(True) for n in ("q", "ql", "k"))
        xx, ws = place(x).requires_grad_(True), [w.float().requires_grad_(True) for w in a.split(16)]
        u = LoRADownDropout.apply(xx, (0.3, 0.1), _rng(), 1, BF16, *ws)
        outs = (u, *QKNormRope.apply(q, ql, k, s["wq"], s["wk"], s["eps"], s["cos"], s["sin"]),
                *AxesRope.apply(q, ql, k, pos, inv, (20, 12)))
        for o in outs:
            o.register_hook(lambda g: seen.append(0 if g is None else g.data_ptr() % 16))
        grads = (du, s["gq"], s["gk"], s["gq"], s["gk"])
        for o, g in zip(outs, grads):
            if join:    # the slice of the cat's gradient that goes to o starts 6 bytes behind a boundary
                torch.cat([first, o.reshape(-1)]).backward(torch.cat([first, g.reshape(-1)]), retain_graph=True)
            else:
                o.backward(g.reshape(o.shape), retain_graph=True)
        return [o.detach() for o in outs] + [t.grad for t in (xx, *ws, q, ql, k)]

    want = run(lambda t: t.detach().clone(memory_format=torch.contiguous_format), False)
    seen.clear()
    got = run(off, True)
    assert 6 in seen
    assert all(torch.equal(a_, b_) for a_, b_ in zip(got, want))
    wide = torch.zeros(20, 131, dtype=BF16, device="cuda")
    wide[:, 3:] = x
    assert torch.equal(LoRADownDropout.apply(wide[:, 3:], (0.3, 0.1), _rng(), 1, BF16, *a.float().split(16)), want[0])


def test_second_derivatives_are_refused(ops):
    """The backward passes are kernels of their own without a derivative: to differentiate them again raises,
    it does not leave the terms out."""
    from decik_b200.solution.attn import AxesRope, QKNormRope
    from decik_b200.solution.dropout import CounterDropout, LoRADownDropout

    s = _heads_case(20, 4, 2, 64, 64, BF16)
    inv, pos = torch.rand(32, device="cuda"), torch.randint(0, 500, (2, 20), device="cuda")
    x, a, _, _ = _lora_case(20, 64, 16, (0.3,), FP32, BF16)
    leaf = lambda t: t.detach().clone().requires_grad_(True)
    for fn, t in ((lambda t: CounterDropout.apply(t, 0.3, _rng()), x),
                  (lambda t: LoRADownDropout.apply(t, 0.3, _rng(), 0, BF16, a.float()), x),
                  (lambda t: QKNormRope.apply(t, None, s["k"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])[0], s["q"]),
                  (lambda t: AxesRope.apply(t, None, s["k"], pos, inv, (20, 12))[0], s["q"])):
        t = leaf(t)
        y = fn(t)
        g, = torch.autograd.grad((y.float() ** 2).sum(), t, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (g.float().sum() + (t.float() ** 2).sum()).backward()


def test_captured_step_draws_new_masks(ops):
    """One captured forward and backward: replays read the generator's state from the device."""
    from decik_b200.solution.dropout import CounterRNG

    r = CounterRNG(9)
    x, a, du, add = _lora_case(64, 256, 16, (0.5, 0.5), FP32, BF16)

    def step():
        s = r.take(3)
        x16, u = ops.lora_down_dropout(x, a, (0.5, 0.5), s)
        dx, da = ops.lora_down_dropout_bwd(du, x16, a, (0.5, 0.5), s, addend=add)
        return u, dx, da, ops.dropout(x, 0.5, s, 2)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    r.state[1] = 0
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):   # a second graph with workspaces of its own
        out2 = step()
    for k in range(4):
        (graph, other)[k % 2].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, out2)[k % 2]]
        state = torch.tensor([9, 3 * k], device="cuda")
        x16, u = ops.lora_down_dropout(x, a, (0.5, 0.5), state)
        dx, da = ops.lora_down_dropout_bwd(du, x16, a, (0.5, 0.5), state, addend=add)
        for a_, b_ in zip(got, (u, dx, da, ops.dropout(x, 0.5, state, 2))):
            assert torch.equal(a_, b_)


def test_captured_training_step(ops):
    """Forward and backward of the autograd Functions captured once, replayed with the state advancing."""
    from decik_b200.solution.attn import QKNormRope
    from decik_b200.solution.dropout import CounterDropout, CounterRNG, LoRADownDropout

    s = _heads_case(96, 4, 2, 64, 64, BF16)
    leaf = lambda t: t.detach().clone().requires_grad_(True)
    q, k, wq, wk = (leaf(s[n]) for n in ("q", "k", "wq", "wk"))
    x, a = leaf(torch.randn(96, 256, device="cuda")), leaf(torch.randn(16, 256, device="cuda"))
    leaves = [q, k, wq, wk, x, a]
    r = CounterRNG(4)

    def step():
        state = r.take(2)
        oq, ok = QKNormRope.apply(q, None, k, wq, wk, 1e-6, s["cos"], s["sin"])
        u = LoRADownDropout.apply(CounterDropout.apply(x, 0.3, state, 0), (0.5,), state, 1, BF16, a)
        return torch.autograd.grad((oq * oq).float().sum() + ok.float().sum() + (u * u).float().sum(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        r.state.copy_(torch.tensor([4, 10 * i], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        r.state.copy_(torch.tensor([4, 10 * i], device="cuda"))
        for g, w in zip(got, step()):
            assert torch.equal(g, w)
        if i:
            assert not torch.equal(got[4], last)
        last = got[4]


def test_binding_argument_errors(ops):
    """What is no tensor, or not as many arguments, is an error and not a crash."""
    from decik_b200 import _lib

    x, rng = torch.randn(8, device="cuda"), _rng()
    with pytest.raises(RuntimeError, match="not a tensor"):
        ops.dropout([1.0], 0.1, rng)
    with pytest.raises(RuntimeError, match="arguments instead of"):
        _lib.bind().dropout(x, 0.1, rng)
    with pytest.raises((TypeError, RuntimeError)):
        ops.dropout(x, "a", rng)
    with pytest.raises(RuntimeError, match="out_dtype"):
        ops.dropout(x, 0.1, rng, out_dtype=3)
    with pytest.raises(RuntimeError, match="p for each"):
        ops.lora_down_dropout(x.view(1, 8), x.view(1, 8).to(BF16), (0.1, 0.1, 0.1), rng)


def test_two_streams_at_once(ops):
    s = _heads_case(3000, 12, 2, 128, 128, BF16)
    x, a, du, add = _lora_case(3000, 512, 16, (0.1, 0.1), FP32, BF16)
    args = (s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["eps"], s["cos"], s["sin"])
    x16 = x.to(BF16)

    def both():
        return ops.qk_norm_rope_bwd(*args) + ops.lora_down_dropout_bwd(du, x16, a, (0.1, 0.1), rng, addend=add)

    rng = _rng()
    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a_, b_) for a_, b_ in zip(g, want))
