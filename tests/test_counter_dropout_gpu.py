"""Counter-based LoRA dropout in the attention block and through the patched model.

The block's bar is the one of tests/tolerance.py (rel-L2 5e-3, max-abs 2e-2) in fp16. In bf16 its
gradients pass through five roundings of at most 2^-9 each (dO, dS, dq, dy, du): rel-L2 5 * 2^-9."""

import pytest
import torch

from oracle import dropout as o_drop
from tests.qlora_stubs import Linear4bit, LoraLayer
from tests.test_block_gpu import _case
from tests.test_model_gpu import _batch, _model, _step, patched_classes  # noqa: F401 (a fixture)
from tests.tolerance import assert_close16

pytestmark = pytest.mark.gpu

SEED, OFFSET, STREAM = 77, 2 ** 33 + 3, 6


@pytest.fixture()
def counter(cuda_lib):
    """Counter-based dropout switched on for the test, and off again."""
    from decik_b200.solution import dropout

    dropout.use_counter_dropout(123)
    yield dropout
    dropout.use_counter_dropout(False)


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("p", [(0.1, 0.3), (0.5, 0.0), (1.0, 0.2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_block_with_dropout_matches_oracle(cuda_lib, dtype, p, normed):
    from oracle import rmsnorm as o_norm
    from oracle.block import block_forward, dequant_torch

    block, packing, cos, sin, h, dout = _case(dtype, lengths=[37, 128, 1, 211, 14], seed=2)
    rng = torch.tensor([SEED, OFFSET], device="cuda")
    w = 1.0 + 0.1 * torch.randn(h.shape[1], generator=torch.Generator().manual_seed(4))
    hg = h.cuda().requires_grad_(True)
    out = block.forward(hg, packing, cos, sin, norm=(w.cuda(), 1e-6) if normed else None, dropout=(*p, rng, STREAM))
    out.backward(dout.cuda())
    torch.cuda.synchronize()
    got = (out.detach().float().cpu(), hg.grad.cpu()) + tuple(q.grad.cpu() for q in block.lora_params())

    r = lambda t: t.detach().float().cpu().to(dtype).float()    # the 16-bit inputs the kernels get
    x_ref = torch.from_numpy(o_norm.forward(h.numpy(), w.numpy(), 1e-6)[0]).float() if normed else h
    x = r(x_ref).requires_grad_(True)
    params = [r(q).requires_grad_(True) for q in block.lora_params()]
    a_q, b_q, a_v, b_v = params
    keep = [torch.from_numpy(o_drop.keep(h.numel(), p[b], SEED, OFFSET, STREAM + b)).view(h.shape).float()
            * o_drop.cut_scale(p[b])[1] for b in (0, 1)]
    wq, wk, wv = (dequant_torch(block.nf4_states[n]).to(dtype).float() for n in ("q", "k", "v"))
    ref_out = block_forward(x, wq, wk, wv, r(block.bias["q"]), r(block.bias["k"]), r(block.bias["v"]), a_q, b_q, a_v,
                            b_v, block.scaling, cos.cpu(), sin.cpu(), packing.spans, block.n_heads, block.n_kv,
                            keep_q=keep[0], keep_v=keep[1])
    ref_out.backward(dout.float())
    dx = torch.from_numpy(o_norm.backward(x.grad.numpy(), h.numpy(), w.numpy(), 1e-6)).float() if normed else x.grad
    ref = (ref_out.detach(), dx, *(q.grad for q in params))
    for name, a, e in zip(("out", "dx", "dA_q", "dB_q", "dA_v", "dB_v"), got, ref):
        bar = 5e-3 if dtype == torch.float16 or name == "out" else 5 * 2.0 ** -9
        assert_close16(a.numpy(), e.numpy(), f"{name} ({dtype}, p {p})", rel_l2=bar)
    if p[0] == 1.0:
        assert not got[2].any() and not got[3].any()    # nothing reaches the q branch
    assert cuda_lib.decik_kernel_error(1) == 0


def test_block_dropout_near_zero_is_the_block(cuda_lib):
    """A p that rounds to no dropout gives the plain block's result: the same x16 and u to fp32 sums."""
    block, packing, cos, sin, x, dout = _case(torch.float16, lengths=[100, 29], seed=3)
    rng = torch.tensor([1, 2], device="cuda")
    a = block.forward(x.cuda(), packing, cos, sin).detach().float()
    b = block.forward(x.cuda(), packing, cos, sin, dropout=(1e-7, 1e-7, rng, 0)).detach().float()
    # u may round to a neighbouring fp16 value: half a step of it against the whole projection
    assert (a - b).abs().max() <= 2.0 ** -10 * a.abs().max()


def test_rng_advanced_before_backward_is_refused(cuda_lib):
    """The state is read again in backward: autograd refuses it if it was changed in place."""
    block, packing, cos, sin, x, dout = _case(torch.float16, lengths=[33], seed=3)
    rng = torch.tensor([1, 2], device="cuda")
    out = block.forward(x.cuda().requires_grad_(True), packing, cos, sin, dropout=(0.1, 0.1, rng, 0))
    rng[1] += 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward(dout.cuda())


def test_patched_model_takes_the_fused_node_with_dropout(counter, cuda_lib, patched_classes):  # noqa: F811
    """LoRA dropout through the patched model with the switch on: every layer runs as the fused node, the
    same state gives the same loss, the next step another, and torch's generators are left alone."""
    from decik_b200 import solution
    from decik_b200.solution import _state, attn

    dtype, batch = torch.bfloat16, _batch("cuda", [120, 33, 64])
    model = _model("cuda", dtype, 0.1)
    solution.apply(linear4bit_cls=Linear4bit, lora_classes=(LoraLayer,))
    calls, orig = [], attn.FusedAttentionBlock.forward
    try:
        attn.FusedAttentionBlock.forward = staticmethod(lambda ctx, *a: (calls.append(a[-1]), orig(ctx, *a))[1])
        torch.manual_seed(5)
        before = torch.cuda.get_rng_state()
        l0, g0, packed = _step(model, batch, _state.STATE, dtype)
        torch.manual_seed(5)
        assert torch.equal(torch.cuda.get_rng_state(), before)
        l1, _, _ = _step(model, batch, _state.STATE, dtype)
        counter.use_counter_dropout(123)                        # the state starts again
        l2, g2, _ = _step(model, batch, _state.STATE, dtype)
    finally:
        attn.FusedAttentionBlock.forward = orig
    n = len(model.model.layers)
    assert packed and len(calls) == 3 * n and all(c is not None for c in calls)
    assert [c[3] for c in calls[:n]] == [2 * i for i in range(n)]           # streams of their own
    assert calls[0][2].tolist() == [123, 0] and calls[n][2].tolist() == [123, counter.STREAMS]
    assert l0 == l2 and l0 != l1
    assert all(torch.isfinite(g).all() and g.any() for g in g0.values())
    for name in g0:     # the attention backward's fp32 reductions have no fixed order
        assert (g0[name] - g2[name]).norm() <= 1e-2 * g0[name].norm(), name
    # dropout changes the loss a little: the branches are small beside the frozen projections
    off, _, _ = _step(_model("cuda", dtype, 0.0), batch, _state.STATE, dtype)
    assert 0 < abs(off - l0) < 0.05 * off
    assert _state.STATE.dropout is None


def test_dropout_module_on_the_packed_path(counter, cuda_lib, patched_classes):  # noqa: F811
    """nn.Dropout of a packed [1, T, W] tensor draws from the step's streams."""
    from decik_b200 import solution
    from decik_b200.solution import _state
    from decik_b200.solution.varlen import _PackedStep, packing_from_lengths

    solution.apply(linear4bit_cls=Linear4bit, lora_classes=(LoraLayer,))
    drop = torch.nn.Dropout(0.25).train()
    x = torch.ones(1, 40, 16, device="cuda")
    with _PackedStep(packing_from_lengths([30, 10], "cuda")):
        y0, y1 = drop(x), drop(x)
        assert _state.STATE.dropout.next == 2
    for i, y in enumerate((y0, y1)):
        kept = torch.from_numpy(o_drop.keep(640, 0.25, 123, 0, i)).view(1, 40, 16)
        assert torch.equal(y.cpu() != 0, kept) and (y.cpu()[kept] - 4 / 3).abs().max() <= 2.0 ** -23
    z = drop(x[:, :5])      # not the packed sequence: torch's own
    assert z.shape == (1, 5, 16)


def _with_lora(model, ranks, alphas, p):
    """The model's q and v adapters replaced by ones of these ranks and scalings."""
    torch.manual_seed(3)
    for layer in model.model.layers:
        a = layer.self_attn
        for name, r, alpha in zip(("q_proj", "v_proj"), ranks, alphas):
            setattr(a, name, LoraLayer(getattr(a, name).base_layer, r, alpha, p, "cuda"))
    return model


@pytest.mark.parametrize("ranks,alphas,fused,way", [
    ((16, 16), (32, 32), True, "fused"), ((16, 16), (32, 32), False, "pair"), ((16, 16), (32, 16), True, "pair"),
    ((8, 8), (16, 16), True, "pair"), ((32, 32), (32, 32), True, "pair"), ((64, 64), (64, 64), True, "single"),
    ((8, 24), (16, 24), True, "single"), ((4, 4), (8, 8), True, "modules"), ((72, 16), (72, 16), True, "modules")])
def test_every_layer_draws_from_the_counter(counter, cuda_lib, patched_classes, monkeypatch, ranks, alphas, fused,  # noqa: F811
                                            way):
    """With the switch on, layers that the fused node is not for draw from the step's streams too: torch's
    generators stay as they were, and the state alone decides the loss."""
    from decik_b200 import solution
    from decik_b200.solution import _state, attn
    from decik_b200.solution import dropout as drop

    monkeypatch.setenv("SKC_FUSED_BLOCK", "1" if fused else "0")
    dtype, batch = torch.bfloat16, _batch("cuda", [120, 33, 64])
    model = _with_lora(_model("cuda", dtype, 0.1), ranks, alphas, 0.1)
    solution.apply(linear4bit_cls=Linear4bit, lora_classes=(LoraLayer,))
    calls = {"block": [], "down": [], "drop": [], "torch": []}

    def counted(name, fn, pick=lambda a: None):
        return lambda *a, **k: (calls[name].append(pick(a)), fn(*a, **k))[1]

    monkeypatch.setattr(attn.FusedAttentionBlock, "forward",
                        staticmethod(counted("block", attn.FusedAttentionBlock.forward)))
    # ctx, x, p, rng, stream, ...
    monkeypatch.setattr(drop.LoRADownDropout, "forward",
                        staticmethod(counted("down", drop.LoRADownDropout.forward, lambda a: a[4])))
    monkeypatch.setattr(drop.CounterDropout, "forward",
                        staticmethod(counted("drop", drop.CounterDropout.forward, lambda a: a[4])))
    monkeypatch.setattr(attn.LoRAPairFromNorm, "forward",
                        staticmethod(counted("torch", attn.LoRAPairFromNorm.forward)))
    torch.manual_seed(5)    # as the step seeds them
    before = torch.get_rng_state(), torch.cuda.get_rng_state()
    l0, g0, packed = _step(model, batch, _state.STATE, dtype)
    assert torch.equal(torch.get_rng_state(), before[0]) and torch.equal(torch.cuda.get_rng_state(), before[1])
    n = len(model.model.layers)
    assert packed and not calls["torch"]
    want = {"fused": (n, [], []), "pair": (0, [2 * i for i in range(n)], []), "single": (0, list(range(2 * n)), []),
            "modules": (0, [], list(range(2 * n)))}[way]
    assert (len(calls["block"]), calls["down"], calls["drop"]) == want
    l1, _, _ = _step(model, batch, _state.STATE, dtype)
    counter.use_counter_dropout(123)                        # the state starts again
    l2, g2, _ = _step(model, batch, _state.STATE, dtype)
    assert l0 == l2 and l0 != l1
    for name in g0:     # the attention backward's fp32 reductions have no fixed order
        assert torch.isfinite(g0[name]).all() and g0[name].any()
        assert (g0[name] - g2[name]).norm() <= 1e-2 * g0[name].norm(), name
    assert _state.STATE.dropout is None


@pytest.mark.parametrize("ranks", [(8, 8), (32, 32), (24, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_lora_branches_under_the_counter_match_the_oracle(cuda_lib, dtype, ranks):
    """The branches' outputs and gradients against 64 bits. 16-bit roundings: u, the product with B and its
    scaling; backward the scaled gradient, du and (dB) the product; the rest are fp32 sums (2^-23 of each
    term on the tensor cores). All bounds count them against the sums of the terms' magnitudes."""
    import numpy as np

    from decik_b200.solution import attn, dropout
    from decik_b200.solution._state import STATE

    T, W, N, p, scalings = 90, 136, 48, (0.25, 0.0), (2.0, 0.75)
    gen = torch.Generator().manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=gen)
    leaf = lambda t: t.cuda().requires_grad_(True)
    x = leaf(rn(1, T, W))
    a, b = [leaf(rn(r, W) / W ** 0.5) for r in ranks], [leaf(rn(N, r) / r ** 0.5) for r in ranks]
    g = [rn(1, T, N).to(dtype) for _ in ranks]
    flags = torch.backends.cuda.matmul
    saved = flags.allow_fp16_reduced_precision_reduction, flags.allow_bf16_reduced_precision_reduction
    flags.allow_fp16_reduced_precision_reduction = flags.allow_bf16_reduced_precision_reduction = False
    STATE.dropout = dropout.StepStreams(torch.tensor([SEED, OFFSET], device="cuda"))
    try:
        out = attn._lora_counter(x, *[(a[i], b[i], scalings[i], p[i]) for i in (0, 1)], dtype)
        torch.autograd.backward(out, [t.cuda() for t in g])
    finally:
        STATE.dropout = None
        flags.allow_fp16_reduced_precision_reduction, flags.allow_bf16_reduced_precision_reduction = saved
    f64 = lambda t: t.detach().to(dtype).double().cpu().numpy()   # the 16-bit values that the products get
    half, u23 = torch.finfo(dtype).eps / 2, 2.0 ** -23
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0          # half a subnormal step of fp16, per rounding
    x16 = f64(x)[0]
    dx, mdx = np.zeros((T, W)), np.zeros((T, W))
    for i, r in enumerate(ranks):
        keep = o_drop.keep(T * W, p[i], SEED, OFFSET, i).reshape(T, W) * o_drop.cut_scale(p[i])[1]
        xm, ai, bi, gi, s = x16 * keep, f64(a[i]), f64(b[i]), f64(g[i])[0], scalings[i]
        u, mu = xm @ ai.T, np.abs(xm) @ np.abs(ai).T
        du, mdu = s * gi @ bi, s * np.abs(gi) @ np.abs(bi)
        dx, mdx = dx + keep * (du @ ai), mdx + keep * (mdu @ np.abs(ai))
        pairs = (("out", out[i][0], s * u @ bi.T, s * mu @ np.abs(bi).T, 3, W + r + 16),
                 ("db", b[i].grad, s * gi.T @ u, s * np.abs(gi).T @ mu, 3, W + T + 16),
                 ("da", a[i].grad, du.T @ xm, mdu.T @ np.abs(xm), 2, N + T + 16))
        for name, got, want, mag, rounds, sums in pairs:
            err = np.abs(got.detach().double().cpu().numpy() - want)
            # (a subnormal rounding of u or du is of values with magnitudes near 1 here: tiny times their count)
            assert (err <= (1.01 * rounds * half + sums * u23) * mag + tiny * 4 * (T + W)).all(), name
    err = np.abs(x.grad[0].double().cpu().numpy() - dx)
    assert (err <= (1.01 * 2 * half + (N + sum(ranks) + 16) * u23) * mdx + tiny * 4 * (T + W)).all()
