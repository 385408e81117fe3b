"""The operators of the attention inputs without a GPU: the generator against published vectors, the
oracles against each other and against differences, and the refusals of the C entry points (argument
checks that fail before any CUDA call)."""

import ctypes

import numpy as np
import pytest
import torch

from decik_b200 import _lib, ops
from oracle import dropout as o_drop
from oracle import head_rope as o_rope


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), "5f6fb709 0d893f64 4f121f81 4f730a48"),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, "5207ddc2 45165e59 4d8ee751 8c52f662"),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     "4dfccaba 190a87f0 c47362ba b6b5242a")])
def test_philox_published_vectors(counter, key, want):
    """The known answers of Philox4x32-7 that its authors publish with it."""
    got = o_drop.philox(np.asarray([counter], dtype=np.uint64), key)[0]
    assert " ".join(f"{int(v):08x}" for v in got) == want


def test_masks_are_addressed_by_index_and_stream():
    whole = o_drop.keep(4000, 0.3, 5, 2 ** 33 + 1, 3)
    assert np.array_equal(whole[1600:], o_drop.keep(2400, 0.3, 5, 2 ** 33 + 1, 3, start=1600))
    assert np.array_equal(whole, o_drop.keep(4000, 0.3, 5, 2 ** 33 + 4))       # offset + stream
    other = o_drop.keep(4000, 0.3, 5, 2 ** 33 + 1, 4)
    # two streams are independent: they agree with probability .7^2 + .3^2 = .58, sigma 0.0078
    assert abs((whole == other).mean() - 0.58) < 5 * 0.0078
    assert abs(whole.mean() - 0.7) < 5 * (0.21 / 4000) ** 0.5
    assert o_drop.keep(64, 0.0, 1, 1).all() and not o_drop.keep(64, 1.0, 1, 1).any()


@pytest.mark.parametrize("sections,interleaved,want", [
    ((3, 2, 1), False, [0, 0, 0, 1, 1, 2]), ((3, 2, 1), True, [0, 1, 2, 0, 1, 0]), ((0, 4), True, [1, 1, 1, 1]),
    ((24, 20, 20), True, [0, 1, 2] * 20 + [0] * 4)])
def test_axis_of(sections, interleaved, want):
    assert list(ops.rope_axis_of(sections, interleaved)) == want == list(o_rope.axis_of(sections, interleaved))


@pytest.mark.parametrize("sections", [(), (1, 1, 1, 1, 1), (4, -1), (2.5, 1), ("a",), None])
def test_axis_of_refusals(sections):
    with pytest.raises(RuntimeError, match="sections"):
        ops.rope_axis_of(sections)


@pytest.mark.parametrize("normed", [True, False])
def test_head_rope_oracle_gradient(normed):
    """The backward formulas against central differences of the forward, in 64 bits."""
    rng = np.random.default_rng(0)
    T, H, D, R = 3, 2, 32, 16
    x, g = rng.standard_normal((T, H, D)), rng.standard_normal((T, H, D))
    w = 1 + 0.3 * rng.standard_normal(D) if normed else None
    cos, sin = rng.standard_normal((T, R)), rng.standard_normal((T, R))  # any tables, not only rotations
    loss = lambda x, w: (o_rope.forward(x, w, 0.1, cos, sin)[0] * g).sum()
    dx, _, dw, _ = o_rope.backward(g, x, w, 0.1, cos, sin)
    h = 1e-5
    for i in [(0, 0, 0), (1, 1, 7), (2, 0, 9), (2, 1, 20), (0, 1, 31)]:
        e = np.zeros_like(x)
        e[i] = h
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - dx[i]) < 1e-8 * max(1, abs(dx[i])) + 1e-8
        if normed:
            e = np.zeros(D)
            e[i[2]] = h
            assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[i[2]]) < 1e-8 * max(1, abs(dw[i[2]])) + 1e-8


def test_lora_oracle_gradient():
    """dx and dA of the dropped-out down projections against differences (the mask is a constant)."""
    rng = np.random.default_rng(1)
    T, W, r, p = 3, 16, 8, (0.3, 0.6)
    x, a, du = rng.standard_normal((T, W)), rng.standard_normal((2 * r, W)), rng.standard_normal((T, 2 * r))
    loss = lambda x, a: (o_drop.lora_down(x, a, p, 7, 9, 2)[0] * du).sum()
    dx, da, _, _ = o_drop.lora_down_bwd(du, x, a, p, 7, 9, 2)
    h = 1e-5
    for t, k, j in [(0, 0, 0), (1, 5, 3), (2, 15, 15), (1, 9, 8)]:
        e = np.zeros_like(x)
        e[t, k] = h
        assert abs((loss(x + e, a) - loss(x - e, a)) / (2 * h) - dx[t, k]) < 1e-7
        e = np.zeros_like(a)
        e[j, k] = h
        assert abs((loss(x, a + e) - loss(x, a - e)) / (2 * h) - da[j, k]) < 1e-7


def test_counter_dropout_switch(monkeypatch):
    """SKC_COUNTER_DROPOUT: unset or 0 leaves torch's draws, a seed switches the generator on."""
    from decik_b200 import solution
    from decik_b200.solution import _state, attn, dropout, mlp, nf4, rmsnorm, varlen

    for m in (attn, mlp, nf4, rmsnorm, varlen):
        monkeypatch.setattr(m, "patch", lambda *a, **k: None)
    try:
        for value, want in ((None, None), ("0", None), ("", None), ("7", 7)):
            dropout.use_counter_dropout(False)
            monkeypatch.delenv("SKC_COUNTER_DROPOUT", raising=False)
            if value is not None:
                monkeypatch.setenv("SKC_COUNTER_DROPOUT", value)
            solution.apply()
            assert _state.STATE.counter_dropout == want
        streams = dropout.step_streams(torch.device("cpu"))
        assert streams.streams(2)[1] == 0 and streams.streams(1)[1] == 2 and streams.rng.tolist() == [7, 0]
        assert dropout.step_streams(torch.device("cpu")).rng.tolist() == [7, dropout.STREAMS]
        with pytest.raises(RuntimeError, match="more than"):
            streams.streams(dropout.STREAMS)
    finally:
        dropout.use_counter_dropout(False)
    assert dropout.step_streams(torch.device("cpu")) is None


def test_counter_rng_state_is_int64():
    from decik_b200.solution.dropout import CounterRNG

    for seed in (0, 2 ** 63 + 5, -3, 2 ** 64 - 1):
        r = CounterRNG(seed, "cpu")
        assert r.state.tolist()[0] % 2 ** 64 == seed % 2 ** 64
    a, b = r.take(2), r.take(1)
    assert a.tolist()[1] == 0 and b.tolist()[1] == 2 and r.state.tolist()[1] == 3


def test_counter_rng_serves_inference_and_training():
    """Made or advanced inside inference mode, the state goes on outside it, and what was taken can be saved
    for a backward pass."""
    from decik_b200.solution.dropout import CounterRNG

    class Saves(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, state):
            ctx.save_for_backward(state)
            return x * 1

        @staticmethod
        def backward(ctx, grad):
            return grad, None

    with torch.inference_mode():
        r = CounterRNG(7, "cpu")
        first = r.take(3)
    second = r.take(2)
    with torch.inference_mode():
        third = r.take(1)
    assert [t.tolist() for t in (first, second, third)] == [[7, 0], [7, 3], [7, 5]] and r.state.tolist() == [7, 6]
    for state in (first, second, third):
        x = torch.ones(2, requires_grad=True)
        Saves.apply(x, state).sum().backward()
        assert x.grad.tolist() == [1, 1]


def test_functions_align_their_rows():
    """A contiguous tensor that starts off a 16-byte boundary is copied, as are strides that the kernels
    refuse; what they take is passed as it is."""
    from decik_b200.solution.attn import _rows16
    from decik_b200.solution.dropout import _rows

    buf = torch.arange(4 * 2 * 16 + 3, dtype=torch.bfloat16)
    assert buf.data_ptr() % 16 == 0
    for off in (1, 3):
        t = buf[off:off + 128].view(4, 2, 16)
        for got, want in ((_rows16(t), t), (_rows(t.view(8, 16)), t.view(8, 16)), (_rows16(t[:1]), t[:1])):
            assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, want)
    wide = torch.arange(8 * 20.0).view(8, 20)
    for t in (wide[:, 1:17], wide[:1, 2:18].expand(8, 16), wide.bfloat16()[:, 4:20], wide.t(),
              torch.tensor(2.0).expand(8, 16)):
        got = _rows(t)
        assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, t)
    for t in (wide[:, 4:], wide, wide.bfloat16().view(4, 40)[:, 8:24], wide[:1, 4:], wide[0]):
        assert _rows(t) is t
    heads = buf[:128].view(4, 2, 16)
    for t in (heads, heads[:, :1], heads[:, :1].expand(4, 3, 16), heads.transpose(0, 1)):
        assert _rows16(t) is t


@pytest.mark.parametrize("p,ranks", [((0.1, 0.3), (8, 24)), ((0.1, 0.3), (16,)), ((0.1,), (16, 16)), ((), (16,)),
                                     (0.1, (8, 8, 8)), (0.1, ()), ([0.1, 0.1, 0.1], (8, 8)), (0.1, (8, 16))])
def test_lora_down_dropout_function_wants_a_p_for_each_weight(p, ranks):
    """Weights of different ranks, or a number of p's that is not theirs, would get one another's masks."""
    from decik_b200.solution.dropout import LoRADownDropout

    a = [torch.zeros(r, 64) for r in ranks]
    with pytest.raises(RuntimeError, match="LoRADownDropout"):
        LoRADownDropout.apply(torch.zeros(4, 64), p, torch.zeros(2, dtype=torch.int64), 0, torch.bfloat16, *a)


# ------------------------------------------------------------------------------------ refusals
P = ctypes.c_void_p(256)   # never dereferenced: the checks fail before any CUDA call
ODD = ctypes.c_void_p(260)
T3 = _lib.Tensor3
NONE3 = T3(None, 0, 0)


def _v(ts=256, hs=128, ptr=256):
    return T3(ptr, ts, hs)


def _refused(rc, text, code=1):
    assert rc == code, rc
    assert text in _lib.lib().decik_last_error()


@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
def test_dropout_refuses_p(p):
    lib = _lib.lib()
    _refused(lib.decik_dropout(P, 1, None, P, 1, 8, p, P, 0, None), b"not in [0, 1]")
    _refused(lib.decik_lora_down_dropout(P, 2, 64, P, 64, P, 64, P, 32, 32, 4, 64, 16, 2, 0.1, p, P, 0, 1, None),
             b"not in [0, 1]")


def test_dropout_refusals():
    lib = _lib.lib()
    _refused(lib.decik_dropout(P, 3, None, P, 1, 8, 0.1, P, 0, None), b"dtypes")
    _refused(lib.decik_dropout(P, 1, None, P, 1, -1, 0.1, P, 0, None), b"n=-1")
    _refused(lib.decik_dropout(P, 1, None, P, 1, 8, 0.1, None, 0, None), b"null pointer")
    assert lib.decik_dropout(None, 1, None, None, 1, 0, 0.1, None, 0, None) == 0


def test_lora_refusals():
    lib = _lib.lib()
    fwd = lambda x=P, xd=2, ldx=64, ldu=64, uc=32, n=4, w=64, r=16, nb=2, dt=1: lib.decik_lora_down_dropout(
        x, xd, ldx, P, 64, P, 64, P, ldu, uc, n, w, r, nb, 0.1, 0.1, P, 0, dt, None)
    _refused(fwd(w=60), b"width 60")
    _refused(fwd(n=-1), b"T=-1")
    _refused(fwd(r=12), b"rank 12", 3)
    _refused(fwd(r=40), b"rank 40", 3)      # 2 branches of 48 rows
    _refused(fwd(nb=3), b"3 branches", 3)
    _refused(fwd(dt=2), b"dtype 2")
    _refused(fwd(xd=0), b"x of dtype 0")
    _refused(fwd(ldx=56), b"strides shorter")
    _refused(fwd(ldu=24), b"strides shorter")
    _refused(fwd(uc=24), b"u_cols 24")
    _refused(fwd(uc=36), b"u_cols 36")
    _refused(fwd(x=ODD), b"alignment")
    _refused(fwd(ldx=66), b"alignment")
    assert fwd(n=0) == 0
    bwd = lambda du=P, ws=P, da=P, ldx=64, ldd=64, n=4: lib.decik_lora_down_dropout_bwd(
        du, 32, P, ldx, P, 64, None, 0, P, ldd, da, n, 64, 16, 2, 0.1, 0.1, P, 0, 1, ws, None)
    _refused(bwd(du=None), b"null pointer")
    _refused(bwd(ws=None), b"null pointer")
    _refused(bwd(da=None), b"da NULL")
    _refused(bwd(ldx=60), b"strides shorter")
    _refused(bwd(ldd=66), b"alignment")
    _refused(bwd(n=1 << 31), b"T=")
    assert lib.decik_lora_down_dropout_bwd_workspace(0, 64, 16, 2) == 0
    assert lib.decik_lora_down_dropout_bwd_workspace(1000, 64, 16, 2) >= 4 * 64 * 32


def test_norm_rope_refusals():
    lib = _lib.lib()

    def fwd(q=_v(), k=_v(), wq=P, wk=P, wd=2, eps=1e-6, cos=P, n=4, D=128, R=128, dt=1):
        return lib.decik_qk_norm_rope_fwd(q, NONE3, k, wq, wk, wd, eps, cos, P, _v(), _v(), n, 2, 1, D, R, dt, None)

    _refused(fwd(D=120), b"head_dim 120")
    _refused(fwd(D=272), b"head_dim 272")
    _refused(fwd(R=144), b"rotary_dim 144")
    _refused(fwd(R=24), b"rotary_dim 24")
    _refused(fwd(R=0), b"rotary_dim 0")
    _refused(fwd(wq=None), b"NULL norm weight")
    _refused(fwd(wd=5), b"norm weights of dtype 5")
    _refused(fwd(eps=-1.0), b"eps")
    _refused(fwd(eps=float("nan")), b"eps")
    _refused(fwd(cos=None), b"cos / sin")
    _refused(fwd(cos=ODD), b"cos / sin")
    _refused(fwd(q=_v(ptr=264)), b"aligned")
    _refused(fwd(k=_v(ts=252)), b"aligned")
    _refused(fwd(dt=2), b"dtype 2")
    assert fwd(n=0) == 0
    bwd = lambda ws=P, dw=P, gq=_v(): lib.decik_qk_norm_rope_bwd(
        gq, _v(), _v(), NONE3, _v(), P, P, 2, 1e-6, P, P, _v(), _v(), dw, P, 4, 2, 1, 128, 128, 1, ws, None)
    _refused(bwd(ws=None), b"workspace")
    _refused(bwd(ws=ODD), b"workspace")
    _refused(bwd(dw=None), b"dq_weight")
    _refused(bwd(gq=NONE3), b"aligned")


def test_axes_refusals():
    lib = _lib.lib()

    def fwd(pos=P, pd=0, ld=4, axes=3, inv=P, amap=bytes([0, 1, 2, 0] * 16), wq=None, wk=None, n=4, R=128):
        return lib.decik_rope_axes_fwd(_v(), NONE3, _v(), wq, wk, 2, 1e-6, pos, pd, ld, axes, inv, amap, _v(), _v(), n,
                                       2, 1, 128, R, 1, None)

    _refused(fwd(axes=5), b"5 axes")
    _refused(fwd(axes=0), b"0 axes")
    _refused(fwd(pd=2), b"position dtype 2")
    _refused(fwd(pos=None), b"null pointer")
    _refused(fwd(inv=None), b"null pointer")
    _refused(fwd(amap=None), b"null pointer")
    _refused(fwd(ld=3), b"rows of positions")
    _refused(fwd(amap=bytes([0, 1, 3, 0] * 16)), b"frequency 2 has axis 3 of 3")
    _refused(fwd(wq=P), b"for neither")
    _refused(fwd(R=8), b"rotary_dim 8")
    assert fwd(n=0) == 0


@pytest.mark.parametrize("bwd", [False, True])
def test_axes_refuse_an_unaligned_inv_freq(bwd):
    """The kernels read the frequencies in 16-byte pieces: a pointer to the middle of one is refused."""
    tail = (P, 0, 4, 3, ODD, bytes([0, 1, 2, 0] * 16))
    end = (4, 2, 1, 128, 128, 1)
    lib = _lib.lib()
    if bwd:
        rc = lib.decik_rope_axes_bwd(_v(), _v(), _v(), NONE3, _v(), P, P, 2, 1e-6, *tail, _v(), _v(), P, P, *end, None,
                                     None)  # (without a workspace: refused after this check, so that it never runs)
    else:
        rc = lib.decik_rope_axes_fwd(_v(), NONE3, _v(), None, None, 2, 1e-6, *tail, _v(), _v(), *end, None)
    _refused(rc, b"inv_freq is not 16-byte aligned")


@pytest.mark.parametrize("change,text", [
    (dict(u=lambda t: t[:3]), "u contiguous"), (dict(u=lambda t: t[:, :32]), "u contiguous"),
    (dict(u=lambda t: t.half()), "dtype"), (dict(w_cat=lambda t: t.half()), "dtype"),
    (dict(ext_b=lambda t: t.half()), "dtype"), (dict(x16=lambda t: t.float()), "x16 fp16"),
    (dict(x16=lambda t: t[0]), "x16 fp16"), (dict(w_cat=lambda t: t[:511]), "w_cat must be"),
    (dict(w_cat=lambda t: t[:, :128]), "w_cat must be"), (dict(w_cat=lambda t: t.t().contiguous().t()), "w_cat must be"),
    (dict(ext_b=lambda t: t[:511]), "ext_b must be"), (dict(ext_b=lambda t: t[:, :32]), "ext_b must be"),
    (dict(ext_b=lambda t: t.repeat(1, 2)[:, :64]), "ext_b must be"),
    (dict(cos=lambda t: t[:3], sin=lambda t: t[:3]), "cos and sin"), (dict(sin=lambda t: t[:3]), "cos and sin"),
    (dict(cos=lambda t: t.half()), "cos and sin"), (dict(sin=lambda t: t.double()), "cos and sin"),
    (dict(cos=lambda t: t[0]), "cos and sin"), ({}, "CUDA device")])
def test_qkv_proj_gemm_refusals(change, text):
    """Operands of another type or with too few rows, refused on the host before anything is read."""
    T, H, Hq, Hk = 4, 256, 2, 1     # 512 rows of projections
    args = dict(x16=torch.zeros(T, H, dtype=torch.bfloat16), u=torch.zeros(T, 64, dtype=torch.bfloat16),
                w_cat=torch.zeros(544, H, dtype=torch.bfloat16), ext_b=torch.zeros(512, 64, dtype=torch.bfloat16),
                cos=torch.zeros(T, 128), sin=torch.zeros(T, 128))
    args = {n: change.get(n, lambda t: t)(t) for n, t in args.items()}
    with pytest.raises(RuntimeError, match=text):
        ops.qkv_proj_gemm(**args, n_heads=Hq, n_kv=Hk)


def test_entries_refuse_pointers_between_values():
    """A pointer that does not start at a value of its type would be a misaligned access of the kernel."""
    lib, at = _lib.lib(), lambda n: ctypes.c_void_p(256 + n)
    text = b"aligned to"
    drop = lambda x=P, xd=1, res=None, out=P, od=1, rng=P: lib.decik_dropout(x, xd, res, out, od, 8, 0.1, rng, 0, None)
    for kw in (dict(x=at(1)), dict(x=at(2), xd=2), dict(out=at(1)), dict(out=at(2), od=2), dict(res=at(1)),
               dict(res=at(2), od=2), dict(rng=at(4))):
        _refused(drop(**kw), text)
    _refused(lib.decik_lora_down_dropout(P, 2, 64, P, 64, P, 64, P, 32, 32, 4, 64, 16, 2, 0.1, 0.1, at(4), 0, 1, None), text)
    _refused(lib.decik_lora_down_dropout_bwd(P, 32, P, 64, P, 64, None, 0, P, 64, P, 4, 64, 16, 2, 0.1, 0.1, at(4), 0, 1,
                                             P, None), text)
    norm = lambda wq=P, wk=P, wd=2: lib.decik_qk_norm_rope_fwd(_v(), NONE3, _v(), wq, wk, wd, 1e-6, P, P, _v(), _v(), 4, 2,
                                                               1, 128, 128, 1, None)
    for kw in (dict(wq=at(2)), dict(wk=at(2)), dict(wq=at(1), wd=1), dict(wk=at(1), wd=0)):
        _refused(norm(**kw), text)
    bwd = lambda dq=P, dk=P: lib.decik_qk_norm_rope_bwd(_v(), _v(), _v(), NONE3, _v(), P, P, 2, 1e-6, P, P, _v(), _v(), dq,
                                                        dk, 4, 2, 1, 128, 128, 1, P, None)
    _refused(bwd(dq=at(2)), text)
    _refused(bwd(dk=at(1)), text)
    axes = lambda pos, pd: lib.decik_rope_axes_fwd(_v(), NONE3, _v(), None, None, 2, 1e-6, pos, pd, 4, 1, P, bytes(64),
                                                   _v(), _v(), 4, 2, 1, 128, 128, 1, None)
    _refused(axes(at(4), 0), text)
    _refused(axes(at(2), 1), text)


def test_ops_refuse_cpu_tensors():
    q, k = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    w, cs, rng = torch.ones(64), torch.ones(4, 64), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.qk_norm_rope_fwd(q, k, w, w, 1e-6, cs, cs), lambda: ops.dropout(cs, 0.1, rng),
                 lambda: ops.rope_axes_fwd(q, k, torch.zeros(1, 4, dtype=torch.int64), torch.ones(32), (32,)),
                 lambda: ops.lora_down_dropout(cs, q[:, 0], 0.1, rng)):
        with pytest.raises(RuntimeError, match="one CUDA device"):
            call()
