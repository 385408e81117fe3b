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
