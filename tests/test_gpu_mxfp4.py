"""Microscaled 4-bit numbers (``mxfp4_quantize``, ``MXFP4Tensor.dequantize``, ``mxfp4_linear``) against their definition in 64 bits.

Quantised values are exact: equal to the definition's.  A product's bound, elementwise: fp32 sums of the width's products
((width + 8) 2^-24 sum |x||w|) and one rounding to the output's type."""
import pytest
import torch

import cellseg_amd as ca

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TABLE = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def definition(x):
    """-> (values float64 like x, scale bytes [..., blocks])"""
    width = x.shape[-1]
    b = torch.nn.functional.pad(x.double(), (0, -width % 32)).reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(amax)
    power = torch.frexp(torch.where(fine & (amax > 0), amax, 1.0))[1].double() - 1
    s = torch.where(amax > 0, power + 125, 0.0).clamp(min=0)
    scale = torch.exp2(s - 127)
    a = torch.where(fine, b.abs() / scale, 0.0)
    middle = (TABLE[1:] + TABLE[:-1]) / 2
    low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)
    v = torch.copysign(TABLE[torch.where(low % 2 == 0, low, high)], b) * scale
    v = torch.where(fine, v, torch.nan)
    return v.reshape(*x.shape[:-1], -1)[..., :width], torch.where(fine, s, 255.0)[..., 0].to(torch.uint8)


def equal(got, want):
    got, want = got.cpu().double(), want.double()
    return got.shape == want.shape and bool(((got == want) | (got.isnan() & want.isnan())).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (7, 100), (4, 2, 96), (130, 257), (64,), (300, 2048)])
def test_quantise_is_exact(shape, kind):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g))).to(TYPES[kind])
    q = ca.mxfp4_quantize(x.to(DEV))
    values, scales = definition(x)
    assert q.shape == tuple(shape) and q.dtype == x.dtype
    assert torch.equal(q.scales.cpu(), scales)
    assert equal(q.dequantize(torch.float32), values)
    assert equal(q.dequantize(), values.to(x.dtype))                     # fp16 may be too narrow for a value: one rounding


def test_every_border():
    """Every halfway value and its neighbours on both sides, both signs, under small and large scales."""
    middle = ((TABLE[1:] + TABLE[:-1]) / 2).float()
    near = torch.cat([middle, torch.nextafter(middle, torch.tensor(9.0)), torch.nextafter(middle, torch.tensor(-9.0)), TABLE.float(),
                      torch.tensor([5.0, 5.5, 6.5, 7.0, 7.5, 7.999])])
    row = torch.zeros(1, 96)
    row[0, ::32] = 4.5                                                   # puts every block's scale at 1
    at = [i for i in range(96) if i % 32][:len(near)]
    row[0, at] = near
    x = torch.cat([row, -row])
    for shift in (-120, -30, 0, 30, 120):
        y = torch.ldexp(x, torch.tensor(shift))
        q = ca.mxfp4_quantize(y.to(DEV))
        assert equal(q.dequantize(torch.float32), definition(y)[0]), shift


def test_zeros_tiny_huge_and_not_finite():
    x = torch.zeros(8, 64)
    x[1, 3] = 1e-44                                                      # subnormal
    x[2, :32] = 1.5e-38
    x[3] = 3.3e38
    x[4, 5], x[4, 40] = torch.inf, 1.0
    x[5, 33] = torch.nan
    x[6, 0] = -torch.inf
    x[7] = -0.0
    q = ca.mxfp4_quantize(x.to(DEV))
    values, scales = definition(x)
    assert torch.equal(q.scales.cpu(), scales) and equal(q.dequantize(torch.float32), values)
    assert q.codes[4, :16].sum() == 0 and int(q.scales[4, 0]) == 255 and int(q.scales[4, 1]) != 255


def check_linear(x, w, what):
    dtype = x.dtype
    weight = ca.mxfp4_quantize(w.to(DEV))
    y = ca.mxfp4_linear(x.to(DEV), weight)
    xq, wq = definition(x)[0], definition(w)[0]
    want = xq @ wq.t()
    bound = (x.shape[-1] + 8) * 2.0 ** -24 * (xq.abs() @ wq.abs().t()) + torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert y.dtype == dtype and y.shape == want.shape
    over = ((y.cpu().double() - want).abs() / bound.clamp(min=1e-300)).max() if want.numel() else 0
    assert bool(torch.isfinite(y).all()) and over <= 1, f"{what}: {float(over):.3g} of its bound"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,width,outputs", [(1, 1, 1), (1, 32, 16), (1, 100, 130), (1, 2048, 1000), (2, 512, 300), (3, 513, 257), (15, 96, 64), (16, 1024, 48), (17, 700, 129), (40, 2000, 77),
                                                (64, 256, 256), (65, 288, 130), (130, 1056, 300), (300, 640, 520)])
def test_linear(rows, width, outputs, kind):
    g = torch.Generator().manual_seed(rows + width + outputs)
    x = (torch.randn(rows, width, generator=g) * torch.exp(torch.randn(1, width, generator=g))).to(TYPES[kind])
    check_linear(x, torch.randn(outputs, width, generator=g) * torch.exp(torch.randn(outputs, 1, generator=g)), f"{rows}x{width}x{outputs}")


def test_linear_scales_reach_their_own_blocks():
    """Blocks whose scales differ by up to 2^40: a scale applied to another block, row or operand would show by orders of magnitude."""
    for rows, width, outputs in ((1, 1024, 64), (33, 1024, 80), (200, 1600, 300)):
        g = torch.Generator().manual_seed(width)
        size = lambda n: torch.ldexp(torch.ones(n, width // 32), torch.randint(-20, 20, (n, width // 32), generator=g)).repeat_interleave(32, 1)   # noqa: E731
        check_linear(torch.randn(rows, width, generator=g) * size(rows), torch.randn(outputs, width, generator=g) * size(outputs), "scales")


def test_linear_large_tiles():
    g = torch.Generator().manual_seed(1)
    check_linear(torch.randn(3300, 330, generator=g).bfloat16(), torch.randn(4001, 330, generator=g), "large tiles")


def test_linear_strides_and_leading_axes():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(24, 96, generator=g).bfloat16(), torch.randn(50, 96, generator=g)
    weight = ca.mxfp4_quantize(w.to(DEV))
    want = ca.mxfp4_linear(x.to(DEV), weight)
    wide = torch.zeros(24, 300, dtype=torch.bfloat16, device=DEV)
    for off in (0, 1, 8):
        wide[:, off:off + 96] = x.to(DEV)
        assert torch.equal(ca.mxfp4_linear(wide[:, off:off + 96], weight), want)
        assert torch.equal(ca.mxfp4_quantize(wide[:, off:off + 96]).codes, ca.mxfp4_quantize(x.to(DEV)).codes)
    assert torch.equal(ca.mxfp4_linear(x.to(DEV).t().contiguous().t(), weight), want)
    assert torch.equal(ca.mxfp4_linear(x.to(DEV).reshape(2, 3, 4, 96), weight), want.reshape(2, 3, 4, 50))
    assert torch.equal(ca.mxfp4_linear(x.to(DEV)[0], weight), ca.mxfp4_linear(x.to(DEV)[:1], weight)[0])
    shifted = torch.zeros(weight.codes.numel() + 16, dtype=torch.uint8, device=DEV)[5:5 + weight.codes.numel()].view(weight.codes.shape)
    shifted.copy_(weight.codes)
    assert torch.equal(ca.mxfp4_linear(x.to(DEV), ca.MXFP4Tensor(shifted, weight.scales, 96)), want)


def test_linear_no_rows_no_outputs_and_nan():
    w = ca.mxfp4_quantize(torch.randn(20, 64, device=DEV))
    assert ca.mxfp4_linear(torch.zeros(0, 64, device=DEV), w).shape == (0, 20)
    assert ca.mxfp4_linear(torch.zeros(3, 64, device=DEV), ca.mxfp4_quantize(torch.zeros(0, 64, device=DEV))).shape == (3, 0)
    assert ca.mxfp4_quantize(torch.zeros(0, 64, device=DEV)).dequantize().shape == (0, 64)
    x = torch.randn(70, 64, device=DEV)
    x[5, 40] = torch.nan
    for rows in (x, x[5:6]):
        y = ca.mxfp4_linear(rows, w)
        assert torch.isnan(y).any(1).nonzero().flatten().tolist() == [5 if len(rows) > 1 else 0] and torch.isnan(y).sum() == 20
    bad = torch.randn(20, 64, device=DEV)
    bad[3, 0] = torch.inf
    y = ca.mxfp4_linear(torch.randn(70, 64, device=DEV), ca.mxfp4_quantize(bad))
    assert torch.isnan(y[:, 3]).all() and torch.isnan(y).sum() == 70


def test_linear_streams_and_graph():
    x, w = torch.randn(9, 512, device=DEV).bfloat16(), ca.mxfp4_quantize(torch.randn(300, 512, device=DEV))
    want = ca.mxfp4_linear(x, w)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append(ca.mxfp4_linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ca.mxfp4_linear(x, w)
    for seed in range(3):
        x.copy_(torch.randn(9, 512, generator=torch.Generator().manual_seed(seed)))
        eager = ca.mxfp4_linear(x, w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


def test_teacher_in_four_bits_to_a_student():
    """As they are used together: a frozen head in 4 bits gives its top logits, the student's head learns from them and from the targets."""
    g = torch.Generator().manual_seed(4)
    n, v, d, k = 96, 1200, 128, 16
    feature, head = torch.randn(n, d, generator=g).bfloat16(), torch.randn(v, d, generator=g) * 0.2
    hidden, weight = torch.randn(n, d, generator=g), torch.randn(v, d, generator=g) * 0.1
    target = torch.randint(0, v, (n,), generator=g)
    target[:9] = -100
    logits = ca.mxfp4_linear(feature.to(DEV), ca.mxfp4_quantize(head.to(DEV)))
    top = torch.topk(logits.float(), k, dim=1)
    a, b = hidden.to(DEV).requires_grad_(), weight.to(DEV).requires_grad_()
    loss = 0.3 * ca.linear_cross_entropy(a, b, target.to(DEV)) + 0.7 * ca.linear_distillation(a, b, top.indices, top.values, temperature=2.0)
    loss.backward()
    c, e = hidden.double().requires_grad_(), weight.double().requires_grad_()
    z = c @ e.t()
    q = torch.softmax(top.values.cpu().double() / 2, 1)
    kd = 4 * (q * (q.log() - torch.log_softmax(z / 2, 1).gather(1, top.indices.cpu()))).sum(1).mean()
    want = 0.3 * torch.nn.functional.cross_entropy(z, target) + 0.7 * kd
    want.backward()
    # fp32: logits are off by (D + 8) 2^-24 sum|h||w| < 2e-4 at most, losses by twice that, probabilities by that relative to themselves
    ez = (d + 8) * 2.0 ** -24 * float((hidden.abs() @ weight.abs().t()).max())
    assert abs(loss.item() - want.item()) <= 8 * ez + 2.0 ** -15
    size = float(max(weight.abs().max(), hidden.abs().max()))
    assert (a.grad.cpu().double() - c.grad).abs().max() <= (4 * ez + 2.0 ** -14) * 2 * size
    assert (b.grad.cpu().double() - e.grad).abs().max() <= (4 * ez + 2.0 ** -14) * 2 * size


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("width", [1536, 1100, 544])
def test_linear_large_tiles_one_after_the_other(width, kind):
    """324 tiles of 256 x 256 on 256 CUs, so that a block goes from one into the next; several pairs of slabs, that end with the width (1536) or not;
    scales that differ by up to 2^20 from block to block, row to row and output to output."""
    g = torch.Generator().manual_seed(width)
    rows, outputs, blocks = 4400, 4390, -(-width // 32)
    size = lambda n: torch.ldexp(torch.ones(n, blocks), torch.randint(-10, 10, (n, blocks), generator=g)).repeat_interleave(32, 1)[:, :width]   # noqa: E731
    x = (torch.randn(rows, width, generator=g).clamp(-4, 4) * size(rows)).to(TYPES[kind])
    w = torch.randn(outputs, width, generator=g) * size(outputs) / 2 ** 10
    y = ca.mxfp4_linear(x.to(DEV), ca.mxfp4_quantize(w.to(DEV)))
    xq, wq = definition(x)[0].to(DEV), definition(w)[0].to(DEV)
    want = xq @ wq.t()
    bound = (width + 8) * 2.0 ** -24 * (xq.abs() @ wq.abs().t()) + torch.finfo(x.dtype).eps / 2 * 1.01 * want.abs() + (2.0 ** -25 if kind == "fp16" else 0)
    over = float(((y.double() - want).abs() / bound.clamp(min=1e-300)).max())
    assert bool(torch.isfinite(y).all()) and over <= 1, f"{over:.3g} of its bound"
