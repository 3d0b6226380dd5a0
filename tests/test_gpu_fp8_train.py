"""The trainer with 8-bit checkpoints and 8-bit attention projections against the same trainer's ordinary path on the rounded
activations, and against the operators called one by one: equal bit for bit (GPU only)."""
import pytest
import torch

from test_gpu_train import _setup

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _round_tape(tr, tape):
    """Replace what the backward reads by what 8-bit checkpoints of it give back."""
    from mad_amd import ops
    rt = lambda t: None if t is None else ops.unpack_fp8(ops.pack_fp8(t))
    for e, sv in zip(tape["P"]["blocks"], tape["saved"]):
        b = e["spec"]
        sv.x, sv.skip, sv.h = rt(sv.x), rt(sv.skip), rt(sv.h)
        sv.h0 = ops.gn_apply(sv.x, sv.c0, act=True, x2=sv.skip, pool=b.down)
        sv.h1 = ops.gn_apply(sv.h, sv.c1, act=True, drop_seed=sv.seed or 0, drop_p=tr.dropout if sv.seed is not None else 0.0)
        if b.attention:
            sv.y = rt(sv.y)
            sv.hn = ops.gn_apply(sv.y, sv.c2, act=False)
    tape["h_last"] = rt(tape["h_last"])
    tape["hact"] = ops.gn_apply(tape["h_last"], tape["c_out"], act=True)


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
@pytest.mark.parametrize("cfg_file,dropout", [("model_tiny.yaml", 0.0), ("model_tiny.yaml", 0.1), ("model_tiny64.yaml", 0.1)])
def test_checkpoints_give_the_gradients_of_the_rounded_activations(dev, cfg_file, dropout, precision):
    from mad_amd import ops
    from mad_amd.train import UNetTrainer
    runs = []
    for checkpoints in (None, "fp8"):
        _, m, _, x, t, lab, target = _setup(cfg_file, precision, dev, B=3)
        tr = UNetTrainer(m.unet, dropout=dropout, checkpoints=checkpoints)
        tr._drop_calls = 0
        pred, tape = tr.forward(x.to(dev), t.to(dev), lab.to(dev))
        loss, dpred = ops.mse_loss_grad(pred, target.to(dev))
        if checkpoints is None:
            _round_tape(tr, tape)
        else:
            assert all(isinstance(sv.x, ops.Fp8Tensor) and isinstance(sv.h, ops.Fp8Tensor) and sv.h0 is sv.h1 is sv.hn is None
                       for sv in tape["saved"])
        tr.backward(tape, dpred)
        runs.append((pred, loss, {k: v.clone() for k, v in tr.grads.items()}))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    for k, want in runs[0][2].items():
        assert torch.equal(runs[1][2][k], want), k


def test_checkpoints_take_less_memory_and_train(dev):
    from mad_amd.train import UNetTrainer
    peak, losses = {}, {}
    for checkpoints in (None, "fp8"):
        _, m, _, x, t, lab, target = _setup("model_tiny64.yaml", "bf16", dev, B=4)
        tr = UNetTrainer(m.unet, dropout=0.1, checkpoints=checkpoints, products=checkpoints)
        args = [v.repeat(8, *([1] * (v.dim() - 1))).to(dev) for v in (x, t, lab, target)]
        tr.forward_backward(args[0], args[1], args[2], args[3])
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        losses[checkpoints] = float(tr.forward_backward(args[0], args[1], args[2], args[3]))
        peak[checkpoints] = torch.cuda.max_memory_allocated() - base
        before = tr.flat.clone()
        tr.step()
        assert bool(torch.isfinite(tr.flat).all()) and not torch.equal(tr.flat, before)
        del tr, m
    assert peak["fp8"] < 0.75 * peak[None], peak


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_products_are_the_operators(dev, precision):
    """One attention block with 8-bit projections, forward and backward, against the operators called one by one; then two
    accumulated micro-batches."""
    from mad_amd import _lib, ops
    from mad_amd.train import GN_EPS, UNetTrainer
    from mad_amd.unet_spec import gn_groups
    _, m, _, x, t, lab, target = _setup("model_tiny.yaml", precision, dev, B=3)
    tr = UNetTrainer(m.unet, dropout=0.0, products="fp8")
    pred, tape = tr.forward(x.to(dev), t.to(dev), lab.to(dev))
    i, e = next((i, e) for i, e in enumerate(tape["P"]["blocks"]) if e["spec"].attention)
    b, sv = e["spec"], tape["saved"][i]
    co = b.out_channels
    order = torch.arange(3 * co, device=dev).reshape(b.num_heads, 64, 3).permute(0, 2, 1).reshape(-1)
    wq = ops.pack_weight_fp8(tr._param[f"{b.name}.qkv.weight"].view(3 * co, co)[order], transposed=True)
    wp = ops.pack_weight_fp8(tr._param[f"{b.name}.proj.weight"].view(co, co), transposed=True)
    hn = ops.gn_apply(sv.y, sv.c2, act=False)
    qkv, hn8 = ops.linear_fp8(hn, wq, bias=tr._param[f"{b.name}.qkv.bias"][order], save=True)
    att, lse = ops.attention(qkv, b.num_heads, want_lse=True)
    out, att8 = ops.linear_fp8(att, wp, bias=tr._param[f"{b.name}.proj.bias"], residual=sv.y, save=True)
    assert torch.equal(sv.qkv, qkv) and torch.equal(sv.att, att)
    assert torch.equal(tape["saved"][i + 1].x, out)

    g = torch.Generator(device=dev).manual_seed(3)
    dout = (1e-3 * torch.randn(out.shape, generator=g, device=dev)).to(out.dtype)
    dada = torch.zeros_like(tape["ada"])
    tr._block_bwd(e, sv, dout, None, dada, tape["ada"], tape["P"]["aff.total"])
    datt, dwp, dbp = ops.linear_fp8_backward(dout, att8, wp)
    dqkv = ops.attention_backward(qkv, att, datt, lse, b.num_heads)
    dhn, dwq, dbq = ops.linear_fp8_backward(dqkv, hn8, wq)
    want_w, want_b = torch.empty_like(dwq), torch.empty_like(dbq)
    want_w[order], want_b[order] = dwq, dbq
    G = tr.grads
    assert torch.equal(G[f"{b.name}.proj.weight"].view(co, co), dwp) and torch.equal(G[f"{b.name}.proj.bias"], dbp)
    assert torch.equal(G[f"{b.name}.qkv.weight"].view(3 * co, co), want_w) and torch.equal(G[f"{b.name}.qkv.bias"], want_b)
    _, _, dg, db = ops.gn_backward(sv.y, dhn, sv.c2, sv.y_part, e["norm2.g"], e["norm2.b"], gn_groups(co), GN_EPS, act=False, add1=dout)
    assert torch.equal(G[f"{b.name}.norm2.weight"], dg) and torch.equal(G[f"{b.name}.norm2.bias"], db)

    # accumulation adds: twice the same micro-batch is twice its gradient (a power of two: exact), and an update repacks the weights
    args = (x.to(dev), t.to(dev), lab.to(dev), target.to(dev))
    tr.micro_batches = 0
    tr.forward_backward(*args, accumulate=True, last=False)
    once = {k: G[k].clone() for k in (f"{b.name}.proj.weight", f"{b.name}.proj.bias", f"{b.name}.qkv.weight", f"{b.name}.qkv.bias")}
    tr.forward_backward(*args, accumulate=True)
    for k, v in once.items():
        assert torch.equal(G[k], 2 * v), k
    old = tr._weight8(e, "proj.w").q.view(torch.uint8).clone()
    tr.step(lr=1e-2)
    e = tr.unet._pack(dev)["blocks"][i]
    new = tr._weight8(e, "proj.w")
    ref = ops.pack_weight_fp8(tr._param[f"{b.name}.proj.weight"].view(co, co), transposed=True)
    assert torch.equal(new.q.view(torch.uint8), ref.q.view(torch.uint8)) and not torch.equal(new.q.view(torch.uint8), old)


def test_products_and_checkpoints_together_are_deterministic(dev):
    from mad_amd.train import UNetTrainer
    got = []
    for _ in range(2):
        _, m, _, x, t, lab, target = _setup("model_tiny.yaml", "bf16", dev, B=3)
        tr = UNetTrainer(m.unet, dropout=0.1, checkpoints="fp8", products="fp8")
        loss = tr.forward_backward(x.to(dev), t.to(dev), lab.to(dev), target.to(dev))
        got.append((loss, tr.gflat.clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and bool(torch.isfinite(got[0][1]).all())


def _disturb_tape(tr, tape):
    """Every activation that 8-bit checkpoints round, times 1 + an independent uniform disturbance of at most 2^-4."""
    from mad_amd import ops
    g = torch.Generator(device=tape["h_last"].device).manual_seed(5)
    seen = {}                                                 # a block's input may be the skip of another: disturbed once, as it is rounded once

    def rt(t):
        if t is not None and id(t) not in seen:
            seen[id(t)] = (t, (t * (1 + 2.0 ** -4 * (2 * torch.rand(t.shape, generator=g, device=t.device) - 1))).to(t.dtype))
        return None if t is None else seen[id(t)][1]
    for e, sv in zip(tape["P"]["blocks"], tape["saved"]):
        sv.x, sv.skip, sv.h = rt(sv.x), rt(sv.skip), rt(sv.h)
        sv.h0 = ops.gn_apply(sv.x, sv.c0, act=True, x2=sv.skip, pool=e["spec"].down)
        sv.h1 = ops.gn_apply(sv.h, sv.c1, act=True, drop_seed=sv.seed or 0, drop_p=tr.dropout if sv.seed is not None else 0.0)
        if e["spec"].attention:
            sv.y = rt(sv.y)
            sv.hn = ops.gn_apply(sv.y, sv.c2, act=False)
    tape["h_last"] = rt(tape["h_last"])
    tape["hact"] = ops.gn_apply(tape["h_last"], tape["c_out"], act=True)


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
@pytest.mark.parametrize("cfg_file", ["model_tiny.yaml", "model_tiny64.yaml"])
@pytest.mark.parametrize("checkpoints,products", [("fp8", None), (None, "fp8"), ("fp8", "fp8")])
def test_gradients_stay_close_to_the_ordinary_ones(dev, cfg_file, checkpoints, products, precision):
    """The gradients of a step with 8-bit checkpoints, products or both against those of the same step without, block by block.

    Checkpoints: rounding to three fraction bits is off by at most 2^-4 of the element, evenly spread below that.  A uniform disturbance
    of at most 2^-4 of every such element is at least as large in the mean square, and to first order both reach the gradients the
    same way: so the gradients are off by no more than with that disturbance, times 1.5 for the spread of two random draws.
    Products: a rounded operand is off by r = 2^-4 / sqrt(3) of its size in the mean square, and so is its product.  An attention
    block has four operands forward (two of them weights) and four backward; q, k, v and the softmax pass a disturbance on by at most
    its size (scores of about one), and the blocks' residual carries what does not go through them: r * sqrt(8 * blocks) in all."""
    from mad_amd import ops
    from mad_amd.train import UNetTrainer
    runs = []
    for disturb, options in ((False, {}), (True, {}), (False, {"checkpoints": checkpoints, "products": products})):
        _, m, _, x, t, lab, target = _setup(cfg_file, precision, dev, B=3)
        tr = UNetTrainer(m.unet, dropout=0.1, **options)
        tr._drop_calls = 0
        pred, tape = tr.forward(x.to(dev), t.to(dev), lab.to(dev))
        loss, dpred = ops.mse_loss_grad(pred, target.to(dev))
        if disturb:
            _disturb_tape(tr, tape)
        tr.backward(tape, dpred)
        runs.append((pred.double(), {k: v.double().flatten() for k, v in tr.grads.items()}))
    blocks = [e["spec"] for e in tape["P"]["blocks"]]
    attentions = sum(b.attention for b in blocks)
    r = 2.0 ** -4 / 3 ** 0.5
    off = lambda a, b: float((a - b).norm() / b.norm())
    (pred0, want), (_, disturbed), (pred, got) = runs
    if products:
        assert 0 < off(pred, pred0) <= r * (4 * attentions) ** 0.5
    else:
        assert torch.equal(pred, pred0)
    for name in [b.name + "." for b in blocks] + [""]:
        join = lambda d: torch.cat([v for k, v in d.items() if k.startswith(name)])
        bound = (1.5 * off(join(disturbed), join(want)) if checkpoints else 0.0) + (r * (8 * attentions) ** 0.5 if products else 0.0)
        assert 0 < off(join(got), join(want)) <= bound, name
