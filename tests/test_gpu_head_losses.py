"""Losses of a linear head over a large vocabulary (``linear_cross_entropy``, ``linear_distillation``) against their definition in 64 bits.

Tolerances are elementwise bounds, computed beside each result from what the kernels round (u = eps / 2 of the inputs' type):
  z         products of D terms summed in fp32: |dz| <= (D + 8) 2^-24 sum_d |h||w| / T (relative to the scaled logits), at most ``ez``;
  loss      lse and the listed logits move by at most ez each, the exponentials' own error (2^-22 relative, an argument below 2^7 rounded to
            2^-24 of itself: 2^-17) moves lse by 2^-17 at most; T^2 scales all; one rounding to fp32;
  p         relative 2 ez + 2^-16;  G = p - q is rounded once (u, fp16 keeps 2^-24 / 2^14 at least) and q once to fp32;
  dH, dW    those errors through the products' absolute values, fp32 sums of that length, one rounding (u; fp16: 2^-25 at least).
"""
import pytest
import torch

import cellseg_amd as ca

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def make(n, v, d, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, d, generator=g) * spread * d ** -0.5).to(dtype)
    pick = torch.randint(0, v, (n,), generator=g)
    h = (torch.randn(n, d, generator=g) + 1.5 * w[pick].float()).to(dtype)
    return h, w, pick


def teacher(n, v, k, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    return ids, 3 * torch.randn(n, k, generator=g)


class Reference:
    """The definition in float64: losses of the rows, gradients of sum_i weight_i loss_i, and the bounds on what the kernels may be off."""

    def __init__(self, h, w, target=None, ids=None, logits=None, t=1.0, ignore=-100):
        dtype = h.dtype
        self.ug = self.u = unit(dtype)                                   # of the inputs' type; of G, which few rows keep as the sum of two such numbers: u^2
        self.tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        self.h, self.w, self.t = h.double(), w.double(), t
        n, v = h.shape[0], w.shape[0]
        self.q = torch.zeros(n, v, dtype=torch.float64)
        entropy = torch.zeros(n, dtype=torch.float64)
        if target is not None:
            self.live = target != ignore
            self.q[self.live, target[self.live]] = 1.0
        else:
            lg = torch.where(ids >= 0, logits.double(), torch.full_like(logits, -torch.inf, dtype=torch.float64)) / t
            self.live = (lg > -torch.inf).any(1)
            q = torch.nan_to_num(torch.softmax(lg, 1), nan=0.0) * self.live[:, None]
            self.q.scatter_add_(1, ids.clamp(min=0), q)
            entropy = torch.where(q > 0, q * torch.log(q.clamp(min=1e-300)), 0.0).sum(1)
        z = self.h @ self.w.t() / t
        logp = torch.log_softmax(z, 1)
        self.p = logp.exp()
        self.loss = torch.where(self.live, t * t * (entropy - torch.where(self.q > 0, self.q * logp, 0.0).sum(1)), 0.0)
        self.ez = float((h.shape[1] + 8) * 2.0 ** -24 * (self.h.abs() @ self.w.abs().t()).max() / t) if n else 0.0
        self.loss_bound = t * t * (2 * self.ez + 2.0 ** -17) + self.loss.abs() * 2.0 ** -23

    def grads(self, weight):
        """weight [rows]: d / d loss_i.  -> (dH, its bound, dW, its bound)"""
        f = (weight * self.live * self.t)[:, None]
        g = (self.p - self.q) * (f != 0)
        eg = (self.p * (2 * self.ez + 2.0 ** -16) + self.q * 2.0 ** -23 + self.ug * g.abs() + self.tiny * 2.0 ** -14) * (f != 0)
        dh, dw = f * (g @ self.w), (f * g).t() @ self.h
        n, v = g.shape
        bh = f.abs() * ((eg + (v + 64) * 2.0 ** -24 * g.abs()) @ self.w.abs()) + self.u * 1.01 * dh.abs() + 4 * 2.0 ** -24 * dh.abs() + self.tiny
        rows = ((eg + (n + 64) * 2.0 ** -24 * g.abs()) * f.abs()).t() @ self.h.abs()
        if not bool((weight == weight[:1]).all()):                       # a gradient per row is folded into a copy of h: one more rounding
            rows = rows + self.u * ((g * f).abs().t() @ self.h.abs()) + self.tiny * float(f.abs().max() if n else 0) * g.abs().t().sum(1, keepdim=True)
        bw = rows + self.u * 1.01 * dw.abs() + 4 * 2.0 ** -24 * dw.abs() + self.tiny
        return dh, bh, dw, bw


def within(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert over <= 0, f"{what}: {((got - want).abs() / bound).max():.3g} of its bound"


def run_and_check(fn, ref, h, w, reduction, weight=1.0, what=""):
    """fn(hidden, weight, reduction) on the GPU against ``ref``."""
    h, w = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = fn(h, w, reduction)
    assert loss.dtype == torch.float32
    n, count = ref.loss.shape[0], max(1, int(ref.live.sum()))
    if reduction == "none":
        within(loss, ref.loss, ref.loss_bound, what + " losses")
        per = weight * (0.25 + torch.rand(n, generator=torch.Generator().manual_seed(9)))
        grad = per.to(DEV)
        per = per.double()
    else:
        by = count if reduction == "mean" else 1
        within(loss, ref.loss.sum() / by, torch.as_tensor(ref.loss_bound).expand(n).sum() / by + (ref.loss.sum() / by).abs() * 2.0 ** -23, what + " loss")
        grad = torch.tensor(weight, device=DEV)
        per = torch.full((n,), weight / by, dtype=torch.float64)
    gh, gw = torch.autograd.grad(loss, (h, w), grad)
    assert gh.dtype == h.dtype and gw.dtype == w.dtype
    dh, bh, dw, bw = ref.grads(per)
    within(gh, dh, bh, what + " grad of hidden")
    within(gw, dw, bw, what + " grad of weight")
    assert not gh[~ref.live.to(DEV)].any(), what + ": a row that does not count has a gradient"


SIZES = [(1, 1, 1), (1, 2, 8), (2, 300, 64), (3, 257, 33), (16, 1000, 128), (33, 129, 100), (64, 4097, 96), (65, 511, 256), (130, 1025, 72),
         (257, 700, 40), (300, 2500, 264), (5, 20000, 16)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,d", SIZES)
def test_cross_entropy(n, v, d, kind):
    h, w, target = make(n, v, d, TYPES[kind], seed=n + v)
    if n > 2:
        target[torch.rand(n, generator=torch.Generator().manual_seed(3)) < 0.3] = -100
    ref = Reference(h, w, target)
    for reduction in ("mean", "none", "sum"):
        run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), ref, h, w, reduction, 64.0 if kind == "fp16" else 0.7, f"{reduction} {n}x{v}x{d}")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,d,k,t", [(1, 1, 1, 1, 1.0), (2, 300, 64, 5, 2.0), (3, 257, 33, 257, 1.0), (16, 1000, 128, 16, 2.0), (33, 129, 100, 100, 4.0), (64, 4097, 96, 64, 0.5),
                                       (130, 1025, 72, 1024, 3.0), (257, 700, 40, 33, 1.0), (300, 2500, 264, 64, 2.0)])
def test_distillation(n, v, d, k, t, kind):
    h, w, _ = make(n, v, d, TYPES[kind], seed=n + k)
    ids, logits = teacher(n, v, k)
    ref = Reference(h, w, ids=ids, logits=logits, t=t)
    for reduction in ("mean", "none", "sum"):
        run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=t, reduction=r), ref, h, w, reduction,
                      64.0 if kind == "fp16" else 0.7, f"{reduction} {n}x{v}x{d} top {k}")


def test_large_shapes_take_the_large_tiles():
    """Sizes where the 256 x 256 tiles run, ragged on every side, with several pieces of the vocabulary's split sums."""
    h, w, target = make(1030, 13001, 200, torch.bfloat16, seed=5)
    target[::7] = -100
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), Reference(h, w, target), h, w, "mean", 1.0, "1030 rows")
    ids, logits = teacher(1030, 13001, 40)
    run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=2.0, reduction=r),
                  Reference(h, w, ids=ids, logits=logits, t=2.0), h, w, "none", 1.0, "1030 rows distilled")


def test_rows_without_target_or_mass():
    h, w, target = make(40, 600, 64, torch.bfloat16)
    nothing = torch.full((40,), -100)
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, nothing.to(DEV), reduction=r), Reference(h, w, nothing), h, w, "mean", 1.0, "all ignored")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, torch.where(target % 2 == 0, 7, target).to(DEV), ignore_index=7, reduction=r),
                  Reference(h, w, torch.where(target % 2 == 0, 7, target), ignore=7), h, w, "mean", 1.0, "another ignore_index")
    ids, logits = teacher(40, 600, 9)
    ids[3] = -1                                                          # no entry
    logits[4] = -torch.inf                                               # no mass
    ids[5, 2:] = -5
    logits[6, :8] = -torch.inf                                           # one entry left: q = 1
    ids[7, 4], logits[8, 0] = -1, -torch.inf
    for reduction in ("mean", "none"):
        run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=1.5, reduction=r),
                      Reference(h, w, ids=ids, logits=logits, t=1.5), h, w, reduction, 1.0, "entries without mass")


def test_an_id_that_comes_twice():
    h, w, _ = make(30, 500, 64, torch.float32)
    ids, logits = teacher(30, 500, 12)
    ids[:, 5] = ids[:, 0]
    ids[:, 9] = ids[:, 0]
    ids[10] = 499
    dense = torch.softmax(logits.double() / 2.0, 1)
    ref = Reference(h, w, ids=ids, logits=logits, t=2.0)                 # its q joins the entries; the loss keeps each entry's own mass
    assert torch.allclose(ref.q.sum(1), dense.sum(1))
    run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=2.0, reduction=r), ref, h, w, "mean", 1.0, "twice")


def test_masked_rows_may_hold_anything():
    """Infinity and NaN in the hidden state of an ignored row reach neither the loss nor any gradient."""
    h, w, target = make(50, 700, 64, torch.bfloat16)
    target[::5] = -100
    want = Reference(h, w, target)
    bad = h.clone()
    bad[0], bad[5], bad[10] = torch.nan, torch.inf, -torch.inf
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), want, bad, w, "mean", 1.0, "masked NaN")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), want, bad, w, "none", 1.0, "masked NaN")


def test_a_target_out_of_range_is_nan_and_reads_nothing_else():
    h, w, target = make(20, 300, 64, torch.float32)
    for wrong in (300, 2 ** 40, -3):
        t = target.clone()
        t[4] = wrong
        a, b = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        losses = ca.linear_cross_entropy(a, b, t.to(DEV), reduction="none")
        assert torch.isnan(losses[4]) and int(torch.isnan(losses).sum()) == 1
        gh, gw = torch.autograd.grad(losses.sum(), (a, b))
        assert torch.isnan(gh[4]).all() and torch.isnan(gh).sum() == gh.shape[1] and torch.isnan(gw).all()
    ids, logits = teacher(20, 300, 6)
    ids[2, 1] = 300
    losses = ca.linear_distillation(h.to(DEV), w.to(DEV), ids.to(DEV), logits.to(DEV), reduction="none")
    assert torch.isnan(losses[2]) and int(torch.isnan(losses).sum()) == 1


def test_infinite_logits():
    """A word that cannot be (all its logits -inf) has probability 0; NaN in a row that counts shows in its loss alone."""
    h, w, target = make(20, 300, 8, torch.float32)
    h, w = h.abs() + 0.1, w.clone()
    w[7] = -torch.inf
    target[target == 7] = 8
    losses = ca.linear_cross_entropy(h.to(DEV), w.to(DEV), target.to(DEV), reduction="none")
    keep = torch.arange(300) != 7
    ref = Reference(h, w[keep], target - (target > 7).long())
    within(losses, ref.loss, ref.loss_bound, "without word 7")
    h[3, 0] = torch.nan
    losses = ca.linear_cross_entropy(h.to(DEV), w.to(DEV), target.to(DEV), reduction="none")
    assert torch.isnan(losses[3]) and int(torch.isnan(losses).sum()) == 1


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_strides_alignment_and_leading_axes(kind):
    dtype = TYPES[kind]
    h, w, target = make(48, 520, 64, dtype)
    ref = Reference(h, w, target)
    t = target.to(DEV)
    wide = torch.zeros(48, 200, dtype=dtype, device=DEV)
    for off in (0, 3, 8):                                                # a column slice: aligned or not
        wide[:, off:off + 64] = h.to(DEV)
        run_and_check(lambda a, b, r: ca.linear_cross_entropy(_leaf_view(a, wide, off), b, t, reduction=r), ref, h, w, "mean", 1.0,
                      f"columns from {off}")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a.t().contiguous().t(), b.t().contiguous().t(), t, reduction=r), ref, h, w, "mean", 1.0, "transposed")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a.reshape(2, 3, 8, 64), b, t.reshape(2, 3, 8), reduction=r).reshape(()), ref, h, w, "mean", 1.0, "leading axes")
    strided = torch.stack([t, t + 1], 1)[:, 0]
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, strided, reduction=r), ref, h, w, "sum", 1.0, "strided target")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, t.int(), reduction=r), ref, h, w, "sum", 1.0, "32-bit target")
    one = Reference(h[:1].expand(48, 64), w, target)
    a, b = h[:1].to(DEV).requires_grad_(), w.to(DEV)
    loss = ca.linear_cross_entropy(a.expand(48, 64), b, t)
    within(loss, one.loss.mean(), one.loss_bound.mean() + one.loss.mean() * 2.0 ** -23, "one row for all")
    dh, bh, _, _ = one.grads(torch.full((48,), 1 / 48, dtype=torch.float64))
    got = torch.autograd.grad(loss, a)[0]                                # autograd adds 48 rows in the inputs' type: a rounding per addition
    within(got, dh.sum(0, keepdim=True), bh.sum(0, keepdim=True) + 48 * unit(dtype) * dh.abs().sum(0, keepdim=True), "gradient of a broadcast row")


def _leaf_view(a, wide, off):
    """The values of ``a`` at columns off.. of a wider tensor, differentiable."""
    class View(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return wide[:, off:off + 64]

        @staticmethod
        def backward(ctx, g):
            return g
    return View.apply(a)


def test_teacher_types_and_strides():
    h, w, _ = make(24, 400, 64, torch.float32)
    ids, logits = teacher(24, 400, 10)
    for dtype in TYPES.values():
        rounded = logits.to(dtype)
        ref = Reference(h, w, ids=ids, logits=rounded.float(), t=2.0)
        both = torch.stack([rounded, rounded], 1).to(DEV)[:, 0]
        run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.int().to(DEV), both, temperature=2.0, reduction=r), ref, h, w, "mean", 1.0, str(dtype))


def test_no_rows():
    w = torch.randn(100, 16, device=DEV, requires_grad=True)
    h = torch.zeros(0, 16, device=DEV, requires_grad=True)
    for reduction in ("mean", "sum"):
        loss = ca.linear_cross_entropy(h, w, torch.zeros(0, dtype=torch.int64, device=DEV), reduction=reduction)
        gh, gw = torch.autograd.grad(loss, (h, w))
        assert loss.item() == 0.0 and gh.shape == (0, 16) and not gw.any()
    assert ca.linear_cross_entropy(h, w, torch.zeros(0, dtype=torch.int64, device=DEV), reduction="none").shape == (0,)
    assert ca.linear_distillation(h, w, torch.zeros(0, 3, dtype=torch.int64, device=DEV), torch.zeros(0, 3, device=DEV)).item() == 0.0


def test_one_gradient_at_a_time_and_frozen_weights():
    h, w, target = make(40, 900, 64, torch.bfloat16)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    both = torch.autograd.grad(ca.linear_cross_entropy(a, b, t), (a, b))
    assert torch.equal(torch.autograd.grad(ca.linear_cross_entropy(a, b.detach(), t), a)[0], both[0])
    assert torch.equal(torch.autograd.grad(ca.linear_cross_entropy(a.detach(), b, t), b)[0], both[1])
    assert not ca.linear_cross_entropy(a.detach(), b.detach(), t).requires_grad


def test_the_same_call_gives_the_same_bits():
    h, w, target = make(300, 5000, 128, torch.bfloat16)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    first = None
    for _ in range(4):
        loss = ca.linear_cross_entropy(a, b, t)
        got = (loss.detach(),) + torch.autograd.grad(loss, (a, b))
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


def test_gradients_against_differences():
    """Central differences of the kernel's own losses, fp32: step 2^-6, loss error <= ref.loss_bound / step, curvature from float64."""
    h, w, target = make(6, 50, 12, torch.float32)
    ids, logits = teacher(6, 50, 5)
    step = 2.0 ** -6
    for fn, ref in ((lambda a, b: ca.linear_cross_entropy(a, b, target.to(DEV), reduction="sum"), lambda a, b: Reference(a, b, target)),
                    (lambda a, b: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=2.0, reduction="sum"),
                     lambda a, b: Reference(a, b, ids=ids, logits=logits, t=2.0))):
        a, b = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        gh, gw = torch.autograd.grad(fn(a, b), (a, b))
        for x, g, at in ((a, gh, 0), (b, gw, 1)):
            for i, j in ((0, 0), (3, 7), (5, 11)):
                d = torch.zeros_like(x)
                d[i, j] = step
                moved = [fn(a + s * d, b) if at == 0 else fn(a, b + s * d) for s in (1, -1)]
                got = (moved[0].double() - moved[1].double()).item() / (2 * step)
                c = [m.detach().cpu() for m in ((a + d, b, a - d) if at == 0 else (a, b + d, b - d))]
                up, down = (ref(c[0], c[1]), ref(c[2], c[1])) if at == 0 else (ref(c[0], c[1]), ref(c[0], c[2]))
                exact = (up.loss.sum() - down.loss.sum()).item() / (2 * step)
                noise = (up.loss_bound.sum() + down.loss_bound.sum()).item() / (2 * step)
                assert abs(got - exact) <= noise
                dh, bh, dw, bw = ref(h, w).grads(torch.ones(6, dtype=torch.float64))
                curved = abs(exact - (dh, dw)[at][i, j].item())          # what the difference itself is off by
                assert abs(g[i, j].item() - got) <= noise + curved + (bh, bw)[at][i, j].item()


def test_another_stream():
    h, w, target = make(200, 3000, 128, torch.bfloat16)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    loss = ca.linear_cross_entropy(a, b, t)
    want = (loss.detach(),) + torch.autograd.grad(loss, (a, b))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                                    # two calls at once
        with torch.cuda.stream(s):
            loss = ca.linear_cross_entropy(a, b, t)
            got.append((loss.detach(),) + torch.autograd.grad(loss, (a, b)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(want, g))


def test_captured_forward_and_backward_replay():
    h, w, target = make(100, 2000, 64, torch.bfloat16)
    ids, logits = teacher(100, 2000, 8)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    ids, logits = ids.to(DEV), logits.to(DEV)

    def both():
        loss = ca.linear_cross_entropy(a, b, t) + 0.5 * ca.linear_distillation(a, b, ids, logits, temperature=2.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in range(3):
        with torch.no_grad():
            h2, w2, t2 = make(100, 2000, 64, torch.bfloat16, seed=20 + seed)
            a.copy_(h2)
            b.copy_(w2)
            t.copy_(t2)
        eager = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager, out))


def test_modules():
    h, w, target = make(10, 100, 16, torch.float32)
    ids, logits = teacher(10, 100, 4)
    a, b = h.to(DEV), w.to(DEV)
    assert torch.equal(ca.LinearCrossEntropyLoss(ignore_index=3, reduction="sum")(a, b, target.to(DEV)), ca.linear_cross_entropy(a, b, target.to(DEV), ignore_index=3, reduction="sum"))
    assert torch.equal(ca.LinearDistillationLoss(temperature=3.0)(a, b, ids.to(DEV), logits.to(DEV)), ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=3.0))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,d", [(1, 130), (16, 77), (17, 257), (33, 300), (64, 515)])
def test_few_rows_keep_more_of_the_gradient_and_read_any_address(n, d, kind):
    """Up to 64 rows G keeps two roundings' worth of bits; rows of both matrices start at odd addresses; a row that does not count holds NaN."""
    v, dtype = 2100, TYPES[kind]
    h, w, target = make(n, v, d, dtype, seed=n + d)
    if n > 1:
        target[n // 2] = -100
    ref = Reference(h, w, target)
    ids, logits = teacher(n, v, 7)
    ids[0] = -1
    kd = Reference(h, w, ids=ids, logits=logits, t=2.0)
    ref.ug = kd.ug = unit(dtype) ** 2 if kind != "fp32" else unit(dtype)
    ids, logits, target = ids.to(DEV), logits.to(DEV), target.to(DEV)

    def odd(x, off):
        return torch.nn.functional.pad(x, (off, 5 - off))[:, off:off + d]

    bad = h.clone()
    if n > 1:
        bad[n // 2] = torch.nan
    for reduction in ("mean", "none"):
        run_and_check(lambda a, b, r: ca.linear_cross_entropy(odd(a, 3), odd(b, 1), target, reduction=r), ref, bad, w, reduction, 64.0 if kind == "fp16" else 0.7,
                      f"{reduction} {n} x {d}")
        run_and_check(lambda a, b, r: ca.linear_distillation(odd(a, 2), odd(b, 3), ids, logits, temperature=2.0, reduction=r), kd, h, w, reduction,
                      64.0 if kind == "fp16" else 0.7, f"{reduction} {n} x {d} distilled")


def test_few_rows_one_gradient_at_a_time_and_twice():
    h, w, target = make(40, 3000, 256, torch.bfloat16)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    loss = ca.linear_cross_entropy(a, b, t)
    both = torch.autograd.grad(loss, (a, b), retain_graph=True)
    again = torch.autograd.grad(loss, (a, b), retain_graph=True)
    one, other = torch.autograd.grad(loss, a, retain_graph=True)[0], torch.autograd.grad(loss, b)[0]
    frozen = torch.autograd.grad(ca.linear_cross_entropy(a, b.detach(), t), a)[0]
    assert all(torch.equal(x, y) for x, y in zip(both + both + both[:1], again + (one, other, frozen)))


@pytest.mark.parametrize("n,v,d,kind", [(40, 3000, 256, "bf16"), (64, 1500, 96, "fp32"), (100, 1500, 77, "fp32"), (1030, 13001, 72, "fp32")])
def test_scores_that_are_not_kept_are_rebuilt(n, v, d, kind):
    """The C entries without keep_scores: the same loss, gradients within the bounds of the larger rounding."""
    from cellseg_amd import _lib, head_losses
    h, w, target = make(n, v, d, TYPES[kind])
    ref = Reference(h, w, target)
    a, b, t = h.to(DEV), w.to(DEV), target.to(DEV)
    losses = []
    for keep in (0, 1):
        head = head_losses._descriptor(a, b, 0, 1, -100, 1.0, 1, t)
        head.keep_scores = keep
        saved = torch.empty(_lib.lib.cs_head_loss_saved_bytes(head), dtype=torch.uint8, device=DEV)
        ws = torch.empty(max(_lib.lib.cs_head_loss_workspace_bytes(head, x) for x in (0, 3)), dtype=torch.uint8, device=DEV)
        loss, one = torch.empty((), device=DEV), torch.ones((), device=DEV)
        gh, gw = torch.empty_like(a), torch.empty_like(b)
        _lib.check(_lib.lib.cs_head_loss_forward(head, None, loss.data_ptr(), saved.data_ptr(), saved.numel(), ws.data_ptr(), ws.numel(), _lib.stream_ptr()), "forward")
        _lib.check(_lib.lib.cs_head_loss_backward(head, saved.data_ptr(), saved.numel(), one.data_ptr(), 0, gh.data_ptr(), gw.data_ptr(), ws.data_ptr(), ws.numel(),
                                                  _lib.stream_ptr()), "backward")
        dh, bh, dw, bw = ref.grads(torch.full((n,), 1 / n, dtype=torch.float64))
        within(gh, dh, bh, f"hidden, keep {keep}")
        within(gw, dw, bw, f"weight, keep {keep}")
        losses.append(loss)
    assert torch.equal(*losses)


@pytest.mark.parametrize("n,v,d", [(4200, 70001, 64), (64, 2100001, 128), (3, 700, 4098)])
def test_a_vocabulary_of_several_pieces(n, v, d):
    """The backward pass takes a large vocabulary in pieces (here two, the second ragged); the last case is wide instead."""
    h, w, target = make(n, v, d, torch.bfloat16)
    ids = torch.stack([target, (target + v // 2) % v, torch.full_like(target, v - 1)], 1)
    logits = torch.randn(n, 3, generator=torch.Generator().manual_seed(4))
    with torch.device(DEV):
        ref = Reference(h.to(DEV), w.to(DEV), ids=ids.to(DEV), logits=logits.to(DEV))
        dh, bh, dw, bw = ref.grads(torch.full((n,), 1 / n, dtype=torch.float64))
    a, b = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV))
    within(loss, ref.loss.mean().cpu(), (ref.loss_bound.mean() + ref.loss.mean() * 2.0 ** -23).cpu(), "loss")
    gh, gw = torch.autograd.grad(loss, (a, b))
    for got, want, bound, what in ((gh, dh, bh, "hidden"), (gw, dw, bw, "weight")):
        assert ((got.double() - want).abs() <= bound).all(), what


def test_few_rows_captured_and_replayed_in_two_graphs():
    h, w, target = make(20, 2000, 128, torch.bfloat16)
    ids, logits = teacher(20, 2000, 8)
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    ids, logits = ids.to(DEV), logits.to(DEV)

    def ce():
        loss = ca.linear_cross_entropy(a, b, t)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b))

    def kd():
        loss = ca.linear_distillation(a, b, ids, logits, temperature=2.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b))

    with torch.cuda.stream(torch.cuda.Stream()):
        ce(), kd()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, fn in zip(graphs, (ce, kd)):
        with torch.cuda.graph(graph):
            outs.append(fn())
    for seed in range(3):
        with torch.no_grad():
            h2, w2, t2 = make(20, 2000, 128, torch.bfloat16, seed=30 + seed)
            a.copy_(h2)
            b.copy_(w2)
            t.copy_(t2)
        want = ce(), kd()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for pair in zip(want, outs) for x, y in zip(*pair))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,d", [(100, 1500, 77), (128, 600, 333), (40, 900, 7), (129, 700, 65), (90, 300, 63)])
def test_rows_at_any_address(n, v, d, kind):
    """Widths that are no multiple of 16 bytes, and rows that start between them: read as they lie, or copied."""
    h, w, target = make(n, v, d, TYPES[kind], seed=n + d)
    target[::6] = -100
    ids, logits = teacher(n, v, 9)
    ref, kd = Reference(h, w, target), Reference(h, w, ids=ids, logits=logits, t=2.0)
    ids, logits, target = ids.to(DEV), logits.to(DEV), target.to(DEV)
    scale = 64.0 if kind == "fp16" else 0.7
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, torch.nn.functional.pad(b, (1, 2))[:, 1:1 + d], target, reduction=r), ref, h, w, "mean", scale, f"{n}x{v}x{d}")
    run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids, logits, temperature=2.0, reduction=r), kd, h, w, "none", scale, f"{n}x{v}x{d} distilled")


@pytest.mark.parametrize("n,d,kind", [(64, 132, "bf16"), (64, 140, "bf16"), (50, 129, "fp16"), (64, 66, "fp32")])
def test_few_rows_over_several_pieces_add_each_column_once(n, d, kind):
    """Widths that end inside a lane's 16 bytes, two pieces of the vocabulary: the columns that two lanes compute are added to the first piece's sums once."""
    v, dtype = 2100001, TYPES[kind]
    g = torch.Generator(device=DEV).manual_seed(d)
    w = (torch.randn(v, d, generator=g, device=DEV) * 2 * d ** -0.5).to(dtype)
    target = torch.randint(0, v, (n,), generator=g, device=DEV)
    target[n // 2:] = v - 1 - torch.arange(n - n // 2, device=DEV)       # half of them in the last piece
    h = (torch.randn(n, d, generator=g, device=DEV) + 1.5 * w[target].float()).to(dtype)
    with torch.device(DEV):
        ref = Reference(h, w, target)
        if kind != "fp32":
            ref.ug = unit(dtype) ** 2
        dh, bh, dw, bw = ref.grads(torch.full((n,), 64.0 / n, dtype=torch.float64))
    a, b = h.requires_grad_(), w.requires_grad_()
    runs = []
    for _ in range(2):
        loss = ca.linear_cross_entropy(a, b, target)
        runs.append(torch.autograd.grad(loss, (a, b), torch.tensor(64.0, device=DEV)))
    for got, want, bound, what in zip(runs[0], (dh, dw), (bh, bw), ("hidden", "weight")):
        assert bool(((got.double() - want).abs() <= bound).all()), what
    assert all(torch.equal(x, y) for x, y in zip(*runs))


@pytest.mark.parametrize("n,d", [(16, 64), (100, 64)])
def test_the_lowest_temperature_and_large_logits(n, d):
    """Logits of several thousand at the lowest temperature, and of 1e8 at temperature 1: |z| / T up to 1e9, where a float's last place is 64."""
    h, w, target = make(n, 500, d, torch.float32)
    ids, logits = teacher(n, 500, 6)
    t = 1e-5
    run_and_check(lambda a, b, r: ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=t, reduction=r), Reference(h * 1000, w, ids=ids, logits=logits, t=t), h * 1000, w,
                  "mean", 1.0, "lowest temperature")
    run_and_check(lambda a, b, r: ca.linear_cross_entropy(a, b, target.to(DEV), reduction=r), Reference(h * 2 ** 24, w, target), h * 2 ** 24, w, "none", 1.0, "large logits")


@pytest.mark.parametrize("n,d,kind", [(1000, 64, "fp32"), (64, 512, "bf16")])
def test_no_scores_are_kept_where_no_backward_pass_can_follow(n, d, kind):
    """Parameters under no_grad and inference_mode: the memory of detached tensors, not that of a training step."""
    v = 16384
    h, w, target = make(n, v, d, TYPES[kind])
    a, b, t = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), target.to(DEV)
    ids, logits = teacher(n, v, 4)
    ids, logits = ids.to(DEV), logits.to(DEV)

    def peak(a, b):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        losses = ca.linear_cross_entropy(a, b, t), ca.linear_distillation(a, b, ids, logits)
        return torch.cuda.max_memory_allocated() - before, losses

    with_scores, want = peak(a, b)
    assert with_scores >= n * v * 4
    alone, got = peak(a.detach(), b.detach())
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            size, got = peak(a, b)
        assert size == alone < n * v * 4
        assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("n,v,d", [(100, 1500, 64), (90, 300, 63), (1030, 13001, 72)])
@pytest.mark.parametrize("distil", [False, True])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_gradients_of_rows_far_apart(n, v, d, distil, kind):
    """16 bits, a gradient per row, from 2^-24 to 1 of the largest: a word that only rows of small gradients name gets its part with all its bits.

    The bound is that of one gradient for all rows: G is rounded once, to u of itself, or in fp16, where it is times its row's factor and 2^14, to 2^-25."""
    h, w, said = make(n, v, d, TYPES[kind], seed=n, spread=8.0)         # each row is sure of one word and wrong: the words it names are its own
    target = (said + 1 + torch.arange(n)) % v
    ids, logits = teacher(n, v, 3)
    size = torch.exp2(-24 * torch.rand(n, generator=torch.Generator().manual_seed(2)))
    size[::9] = 0.0
    size[1] = 1.0
    per = (2048 * size).double()
    with torch.device(DEV):
        ref = Reference(h.to(DEV), w.to(DEV), ids=ids.to(DEV), logits=logits.to(DEV), t=2.0) if distil else Reference(h.to(DEV), w.to(DEV), target.to(DEV))
        f = (per.to(DEV) * ref.t)[:, None]
        g = ref.p - ref.q
        eg = ref.p * (2 * ref.ez + 2.0 ** -16) + ref.q * 2.0 ** -23 + (ref.u + 4 * 2.0 ** -24) * g.abs()
        dw = (f * g).t() @ ref.h
        lost = float(f.max()) * ref.tiny * 2.0 ** -14 * (f != 0)
        rows = (f * (eg + (n + 64) * 2.0 ** -24 * g.abs()) + lost).t() @ ref.h.abs()
        bw = rows + ref.u * 1.01 * dw.abs() + 4 * 2.0 ** -24 * dw.abs() + ref.tiny
    a, b = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    losses = ca.linear_distillation(a, b, ids.to(DEV), logits.to(DEV), temperature=2.0, reduction="none") if distil else ca.linear_cross_entropy(a, b, target.to(DEV), reduction="none")
    gh, gw = torch.autograd.grad(losses, (a, b), per.float().to(DEV))
    over = ((gw.double() - dw).abs() / bw).max().item()
    assert over <= 1, f"grad of weight: {over:.3g} of its bound"
    dh, bh, _, _ = ref.grads(per.to(DEV))
    assert bool(((gh.double() - dh).abs() <= bh).all())
    assert not gh[::9].any()


@pytest.mark.parametrize("n,v,d,kind,distil", [(1531, 32003, 1000, "fp16", False), (1550, 32003, 1000, "bf16", False), (1550, 32003, 1000, "fp16", True), (1531, 32003, 1000, "bf16", True),
                                               (8100, 1500, 4096, "bf16", False), (1000, 16384, 2048, "fp32", False), (2050, 66001, 260, "fp32", True)])
def test_large_tiles_one_after_the_other(n, v, d, kind, distil):
    """More than 256 tiles of 256 x 256, of several slabs each, so that a block goes from one into the next: in the losses, in G (with and without its rows'
    factors) and in both gradients, where k ends inside a slab and where it does not, cut and whole.  Of the 16-bit cases the first four take
    large tiles in all four products, the fifth in the gradient of hidden with k whole; the float32 cases in the losses, and in the gradient of weight (1000
    rows) or in G, from logits that are not kept (2050 rows)."""
    g = torch.Generator(device=DEV).manual_seed(n + d)
    dtype = TYPES[kind]
    w = (torch.randn(v, d, generator=g, device=DEV) * 2 * d ** -0.5).to(dtype)
    target = torch.randint(0, v, (n,), generator=g, device=DEV)
    h = (torch.randn(n, d, generator=g, device=DEV) + 1.5 * w[target].float()).to(dtype)
    with torch.device(DEV):
        if distil:
            ids = torch.stack([target, (target + 1) % v, (target * 7 + 5) % v, torch.full_like(target, v - 1)], 1)
            logits = 2 * torch.randn(n, 4, generator=g)
            ref = Reference(h, w, ids=ids, logits=logits, t=2.0)
            per = 512 * (0.25 + torch.rand(n, generator=g))
        else:
            target[::7] = -100
            ref = Reference(h, w, target)
            per = torch.full((n,), 512.0 / int(ref.live.sum()))
        dh, bh, dw, bw = ref.grads(per.double())
    a, b = h.requires_grad_(), w.requires_grad_()
    if distil:
        loss = ca.linear_distillation(a, b, ids, logits, temperature=2.0, reduction="none")
        assert bool(((loss.double() - ref.loss).abs() <= ref.loss_bound).all())
    else:
        loss = ca.linear_cross_entropy(a, b, target)
        mean = ref.loss.sum() / ref.live.sum()
        assert abs(loss.item() - mean.item()) <= ((ref.loss_bound.sum() / n) + mean * 2.0 ** -23).item()
    gh, gw = torch.autograd.grad(loss, (a, b), per if distil else torch.tensor(512.0, device=DEV))
    for got, want, bound, what in ((gh, dh, bh, "hidden"), (gw, dw, bw, "weight")):
        over = float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max())
        assert bool(torch.isfinite(got).all()) and over <= 1, f"{what}: {over:.3g} of its bound"
