"""Calls of the head losses and of the 4-bit operators that their other tests do not make: rows without a target above 64 rows, rows and widths far apart,
offsets beyond 32 bits, graphs of the larger kernels, tensors saved on the host.  Bounds: those of test_gpu_head_losses.py and test_gpu_mxfp4.py."""
import pytest
import torch

import cellseg_amd as ca
from test_gpu_head_losses import DEV, TYPES, Reference, make, run_and_check, teacher, unit, within
from test_gpu_mxfp4 import definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,d", [(100, 700, 64), (129, 520, 77), (1030, 3001, 72)])
def test_rows_that_do_not_count_may_hold_anything(n, v, d, kind):
    """More than 64 rows: NaN and infinity in rows without a target, or without a teacher's mass, reach neither the loss nor a gradient."""
    h, w, target = make(n, v, d, TYPES[kind], seed=n)
    ids, logits = teacher(n, v, 5)
    target[::5] = -100
    ids[::10] = -1
    logits[5::10] = -torch.inf
    logits[1, :4], ids[2, 1:] = -torch.inf, -7                           # one entry left
    logits[3, 1], ids[4, 0] = torch.finfo(torch.float32).min, -1
    bad = h.clone()
    bad[0::15], bad[5::15], bad[10::15] = torch.nan, torch.inf, -torch.inf
    ids_bad = logits.clone()
    ids_bad[ids < 0] = torch.nan                                         # a logit behind a negative id
    scale = 64.0 if kind == "fp16" else 0.7
    for reduction in ("mean", "none"):
        run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), Reference(h, w, target), bad, w, reduction, scale, "cross entropy")
        run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), ids_bad.to(DEV), temperature=1.5, reduction=r), Reference(h, w, ids=ids, logits=logits, t=1.5), bad, w,
                      reduction, scale, "distillation")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [20, 100, 1030])
def test_ids_out_of_range_make_their_row_nan(n, kind):
    h, w, target = make(n, 3001, 64, TYPES[kind])
    ids, logits = teacher(n, 3001, 6)
    target[4], ids[4, 2] = 3001, 2 ** 33
    a, b = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    for losses in (ca.linear_cross_entropy(a, b, target.to(DEV), reduction="none"), ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), reduction="none")):
        assert torch.isnan(losses).nonzero().flatten().tolist() == [4]
        for grad in (torch.ones(n, device=DEV), torch.linspace(1, 2, n, device=DEV)):
            gh, gw = torch.autograd.grad(losses, (a, b), grad, retain_graph=True)
            assert torch.isnan(gh[4]).all() and int(torch.isnan(gh).sum()) == gh.shape[1] and torch.isnan(gw).all()


@pytest.mark.parametrize("n,v,d,kind", [(200001, 5, 16, "bf16"), (200001, 5, 16, "fp32"), (70, 300, 70001, "fp16"), (70, 300, 70001, "fp32"), (20, 200, 40003, "bf16")])
def test_many_rows_and_long_rows(n, v, d, kind):
    g = torch.Generator(device=DEV).manual_seed(d)
    dtype = TYPES[kind]
    w = (torch.randn(v, d, generator=g, device=DEV) * 2 * d ** -0.5).to(dtype)
    target = torch.randint(0, v, (n,), generator=g, device=DEV)
    h = torch.randn(n, d, generator=g, device=DEV).to(dtype)
    target[::3] = -100
    with torch.device(DEV):
        ref = Reference(h, w, target)
        per = 4 * (0.25 + torch.rand(n, generator=g))
        dh, bh, dw, bw = ref.grads(per.double())
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ca.linear_cross_entropy(a, b, target, reduction="none")
    within(loss, ref.loss.cpu(), ref.loss_bound.cpu(), "losses")
    gh, gw = torch.autograd.grad(loss, (a, b), per)
    within(gh, dh.cpu(), bh.cpu(), "hidden")
    within(gw, dw.cpu(), bw.cpu(), "weight")


@pytest.mark.parametrize("n", [20, 100])
def test_a_weight_of_more_than_2_to_the_31_values(n):
    """530 000 words of 4096: the 64-bit reference goes over the words in pieces, the gradient of weight is compared where offsets pass 32 bits and at both ends."""
    v, d, piece = 530000, 4096, 53000
    g = torch.Generator(device=DEV).manual_seed(n)
    w = torch.empty(v, d, dtype=torch.bfloat16, device=DEV).normal_(generator=g).mul_(2 * d ** -0.5)
    target = torch.randint(0, v, (n,), generator=g, device=DEV)
    target[0], target[1], target[2] = v - 1, 0, 2 ** 31 // d
    h = (torch.randn(n, d, generator=g, device=DEV) + 1.5 * w[target].float()).bfloat16()
    hd, u = h.double(), unit(torch.bfloat16)
    z = torch.cat([hd @ w[i:i + piece].double().t() for i in range(0, v, piece)], 1)
    ez = (d + 8) * 2.0 ** -24 * max(float((hd.abs() @ w[i:i + piece].double().abs().t()).max()) for i in range(0, v, piece))
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    q = torch.zeros_like(p).scatter_(1, target[:, None], 1.0)
    losses = -logp.gather(1, target[:, None])[:, 0]
    grads = (p - q) / n
    eg = (p * (2 * ez + 2.0 ** -16) + q * 2.0 ** -23) / n + u * grads.abs()
    a, b = h.requires_grad_(), w.requires_grad_()
    loss = ca.linear_cross_entropy(a, b, target)
    assert abs(loss.item() - losses.mean().item()) <= 2 * ez + 2.0 ** -17 + losses.mean().item() * 2.0 ** -22
    gh, gw = torch.autograd.grad(loss, (a, b))
    w, dh, bh = w.detach(), torch.zeros_like(hd), torch.zeros_like(hd)
    for i in range(0, v, piece):
        part = w[i:i + piece].double()
        dh += grads[:, i:i + piece] @ part
        bh += (eg + (v + 64) * 2.0 ** -24 * grads.abs())[:, i:i + piece] @ part.abs()
    assert bool(((gh.double() - dh).abs() <= bh + 1.01 * u * dh.abs()).all())
    for i in (0, 2 ** 30 // d - 300, 2 ** 31 // d - 300, v - 600):
        want = grads[:, i:i + 600].t() @ hd
        bound = (eg + (n + 64) * 2.0 ** -24 * grads.abs())[:, i:i + 600].t() @ hd.abs() + 1.01 * u * want.abs()
        assert bool(((gw[i:i + 600].double() - want).abs() <= bound).all()), i


def test_tensors_saved_on_the_host():
    """Saved tensors that come back from the host lie elsewhere, with other strides."""
    for n, d, kind in ((40, 256, "bf16"), (100, 77, "fp32"), (300, 100, "fp16")):
        h, w, target = make(n, 900, d + 3, TYPES[kind])
        a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
        ref = Reference(h[:, 1:1 + d], w[:, 2:2 + d], target)
        with torch.autograd.graph.save_on_cpu():
            loss = ca.linear_cross_entropy(a[:, 1:1 + d], b[:, 2:2 + d], t)
        gh, gw = torch.autograd.grad(loss, (a, b), torch.tensor(8.0, device=DEV))
        dh, bh, dw, bw = ref.grads(torch.full((n,), 8.0 / n, dtype=torch.float64))
        within(gh[:, 1:1 + d], dh, bh, "hidden")
        within(gw[:, 2:2 + d], dw, bw, "weight")
        assert not gh[:, 0].any() and not gw[:, :2].any()


def test_a_tied_weight_and_a_forward_mode_tangent():
    """Rows of the weight as hidden state get both gradients; the losses refuse a tangent, which they would lose."""
    w = torch.randn(200, 32, generator=torch.Generator().manual_seed(0))
    target = torch.arange(70) + 100
    b = w.to(DEV).requires_grad_()
    got = torch.autograd.grad(ca.linear_cross_entropy(b[:70], b, target.to(DEV)), b)[0]
    ref = Reference(w[:70], w, target)
    dh, bh, dw, bw = ref.grads(torch.full((70,), 1 / 70, dtype=torch.float64))
    dw[:70] += dh
    bw[:70] += bh
    within(got, dw, bw + 2.0 ** -23 * dw.abs(), "both")
    ids, logits = teacher(70, 200, 3)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(b.detach(), torch.ones_like(b))
        for call in (lambda: ca.linear_cross_entropy(b.detach()[:70], dual, target.to(DEV)), lambda: ca.linear_distillation(dual[:70], b.detach(), ids.to(DEV), logits.to(DEV)),
                     lambda: ca.mxfp4_quantize(dual)):
            with pytest.raises((NotImplementedError, ValueError)):
                call()


@pytest.mark.parametrize("rows", [40, 300])
def test_quantisation_and_layer_in_two_graphs(rows):
    """The larger kernels of the 4-bit layer, with their workspaces, and the quantisation of a weight, captured and replayed in turn with eager calls between."""
    x, w = torch.randn(rows, 520, device=DEV).half(), torch.randn(600, 520, device=DEV)

    def layer():
        return ca.mxfp4_linear(x, ca.mxfp4_quantize(w))

    def back():
        return ca.mxfp4_quantize(x).dequantize()

    with torch.cuda.stream(torch.cuda.Stream()):
        layer(), back()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, fn in zip(graphs, (layer, back)):
        with torch.cuda.graph(graph):
            outs.append(fn())
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(rows, 520, generator=g))
        w.copy_(torch.randn(600, 520, generator=g))
        want = layer(), back()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_four_bit_tensors_of_more_than_2_to_the_31_values():
    x = torch.empty(70000, 32768, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    q = ca.mxfp4_quantize(x)
    back = q.dequantize()
    for i in (0, 2 ** 31 // 32768 - 20, 70000 - 40):
        part = ca.mxfp4_quantize(x[i:i + 40])
        assert torch.equal(q.codes[i:i + 40], part.codes) and torch.equal(q.scales[i:i + 40], part.scales)
        values = definition(x[i:i + 40].cpu())[0]
        assert torch.equal(back[i:i + 40].cpu().double(), values)
    del x, q, back
    g = torch.Generator(device=DEV).manual_seed(2)
    x, w = torch.randn(140000, 64, generator=g, device=DEV).bfloat16(), torch.randn(16400, 64, generator=g, device=DEV)
    y = ca.mxfp4_linear(x, ca.mxfp4_quantize(w))
    wq = definition(w.cpu())[0].to(DEV)
    for i in (0, 2 ** 31 // 16400 - 150, 140000 - 300):
        xq = definition(x[i:i + 300].cpu())[0].to(DEV)
        want = xq @ wq.t()
        bound = 72 * 2.0 ** -24 * (xq.abs() @ wq.abs().t()) + 1.01 * unit(torch.bfloat16) * want.abs()
        assert bool(((y[i:i + 300].double() - want).abs() <= bound).all()), i


@pytest.mark.parametrize("n,v,kind", [(40, 900, "bf16"), (100, 900, "fp16"), (1030, 5001, "bf16"), (100, 900, "fp32")])
def test_a_gradient_per_row_captured_and_replayed(n, v, kind):
    """reduction="none" in two graphs, replayed in turn with eager calls on another stream between."""
    h, w, target = make(n, v, 128, TYPES[kind])
    ids, logits = teacher(n, v, 5)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    ids, logits, per = ids.to(DEV), logits.to(DEV), torch.rand(n, device=DEV)

    def ce():
        losses = ca.linear_cross_entropy(a, b, t, reduction="none")
        return (losses.detach(),) + torch.autograd.grad(losses, (a, b), per)

    def kd():
        losses = ca.linear_distillation(a, b, ids, logits, temperature=3.0, reduction="none")
        return (losses.detach(),) + torch.autograd.grad(losses, (a, b), per)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ce(), kd()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, fn in zip(graphs, (ce, kd)):
        with torch.cuda.graph(graph):
            outs.append(fn())
    for seed in range(3):
        with torch.no_grad():
            h2, w2, t2 = make(n, v, 128, TYPES[kind], seed=40 + seed)
            a.copy_(h2)
            b.copy_(w2)
            t.copy_(torch.where(torch.rand(n, generator=torch.Generator().manual_seed(seed)) < 0.2, -100, t2))
            per.copy_(torch.exp2(-20 * torch.rand(n, generator=torch.Generator().manual_seed(seed))))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = ce(), kd()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for pair in zip(want, outs) for x, y in zip(*pair))
