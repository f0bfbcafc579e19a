"""4-bit products where the sum itself is exact, so that nothing but the last rounding may be off; and their mean error in fp32."""
import math

import pytest
import torch

from oracle import decode as O
from tts_amd import ops

from .test_decode_gpu import F, TYPES, _g, _within, u

pytestmark = pytest.mark.gpu

# rows, outputs, k, group: few rows and many, one, two and four tiles of outputs a workgroup, chunks of 128 in part
SHAPES = [(1, 40, 4096, 64), (1, 20, 96, 32), (4, 33, 1024, 128), (5, 8200, 192, 64), (6, 50, 640, 32), (16, 100, 2048, 128), (17, 8200, 256, 32), (40, 16400, 128, 64), (3, 8195, 160, 32)]


@pytest.mark.parametrize("m,n,k,group", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_levels_at_the_zero_point_weigh_nothing(gpu, dtype, m, n, k, group):
    """Weights of zero give the bias, whatever x holds and wherever the zero point lies."""
    g = _g(k + m)
    x = torch.randn(m, k, generator=g).to(dtype)
    x[0] = x[0].abs() * 100                                   # a sum of x far from zero
    bias = torch.randn(n, generator=g).to(dtype)
    s = torch.rand(n, k // group, generator=g).to(dtype) + 1
    for zeros in (None, torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)):
        z = torch.full((n, k // group), 8, dtype=torch.uint8) if zeros is None else zeros
        q = z.repeat_interleave(group, 1)
        up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
        got = ops.linear_w4(ops.PackedW4(up(q[:, ::2] | q[:, 1::2] << 4), up(s), up(zeros), up(bias)), up(x))
        assert torch.equal(got.cpu(), bias.expand(m, n)), "%d of %d values off, worst %g" % (
            int((got.cpu() != bias).sum()), m * n, float((got.cpu().float() - bias.float()).abs().max()))


@pytest.mark.parametrize("m,n,k,group", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_single_weight_gives_its_product(gpu, dtype, m, n, k, group):
    """One level off the zero point an output, by a power of two: x itself, scaled, to its last bit (in fp32 every part of it)."""
    g = _g(k + n)
    x = torch.randn(m, k, generator=g).to(dtype)
    q = torch.full((n, k), 8, dtype=torch.uint8)
    at, off = torch.randint(0, k, (n,), generator=g), torch.tensor([-8, -4, -2, -1, 1, 2, 4])[torch.randint(0, 7, (n,), generator=g)]
    q[torch.arange(n), at] = (8 + off).to(torch.uint8)
    s = torch.full((n, k // group), 0.25, dtype=dtype)
    got = ops.linear_w4(ops.PackedW4((q[:, ::2] | q[:, 1::2] << 4).to(gpu), s.to(gpu)), x.to(gpu)).cpu()
    want = (x[:, at].double() * off * 0.25).to(dtype)
    assert torch.equal(got, want), "%d of %d values off" % (int((got != want).sum()), m * n)


@pytest.mark.parametrize("levels", ["even", "bell", "sparse"])
@pytest.mark.parametrize("m,n,k,group", [(1, 64, 4096, 64), (5, 64, 4096, 128), (24, 64, 4096, 32), (3, 64, 8192, 128)])
def test_fp32_error_is_that_of_fp32_sums(gpu, m, n, k, group, levels):
    """Root mean square over the outputs, relative to sum |x w|: within twice that of plain fp32 products summed one after the other a
    hundred and twenty-eight at a time (both are sums of some k / 128 and 128 roundings of partial sums; the products here are exact)."""
    g = _g(m + k)
    x = torch.randn(m, k, generator=g)
    q = {"even": torch.randint(0, 16, (n, k), generator=g), "bell": (8 + 2.5 * torch.randn(n, k, generator=g)).round().clamp(0, 15),
         "sparse": torch.where(torch.rand(n, k, generator=g) < 0.98, 8, torch.randint(0, 16, (n, k), generator=g))}[levels].to(torch.uint8)
    s = torch.rand(n, k // group, generator=g) + 0.5
    packed = q[:, ::2] | q[:, 1::2] << 4
    got = ops.linear_w4(ops.PackedW4(packed.to(gpu), s.to(gpu)), x.to(gpu)).cpu().double()
    want, mag = O.linear_w4(x, packed, s)
    w = (q.float() - 8) * s.repeat_interleave(group, 1)
    plain = torch.zeros(m, n)
    for c in range(0, k, 128):
        part = torch.zeros(m, n)
        for j in range(c, c + 128):
            part = part + x[:, j: j + 1] * w[None, :, j]
        plain = plain + part
    rms = lambda y: float((((y.double() - want) / mag) ** 2).mean().sqrt())  # noqa: E731
    assert rms(got) <= 2 * rms(plain), "%.3g, plain %.3g" % (rms(got), rms(plain))


def test_fp32_rows_whose_large_parts_cancel(gpu):
    """x and its negative but for its last bits, against equal weights: what is left lies in the smaller parts alone."""
    g = _g(1)
    for m, k in ((1, 256), (5, 4096), (24, 512)):
        a = (torch.rand(m, k // 2, generator=g) + 1) * torch.randint(0, 2, (m, k // 2), generator=g).mul(2).sub(1)
        b = -(a.view(torch.int32) ^ torch.randint(0, 1 << 6, a.shape, generator=g, dtype=torch.int32)).view(torch.float32)
        x = torch.stack([a, b], -1).view(m, k)
        n = 40
        q = torch.randint(0, 16, (n, k // 2), generator=g, dtype=torch.uint8)            # both of a byte: one weight for the two
        s = torch.ones(n, k // 64)
        packed = q | q << 4
        got = ops.linear_w4(ops.PackedW4(packed.to(gpu), s.to(gpu)), x.to(gpu))
        want, mag = O.linear_w4(x, packed, s)
        # a partial sum within a product is no larger than the 32 products of it, wherever it is rounded: F of that, sqrt of how many
        _within(got, want, 6 * math.sqrt(3 * k) * F * (32 * 2 * 8.0 + want.abs()), "cancelling")
        rms = float(((got.cpu().double() - want) / mag).pow(2).mean().sqrt())
        assert rms <= 2 * F and float(want.abs().mean()) < 0.05, rms                       # a lost second part is 2^-9 of |x|, a third 2^-17


@pytest.mark.parametrize("m,n,k,group,zeros", [(300, 200, 512, 64, True), (1000, 70, 256, 128, False), (437, 1024, 1024, 64, True), (64, 8192, 1024, 128, False),
                                               (33, 4100, 2080, 32, True), (2, 16400, 256, 64, True), (4, 16400, 384, 128, False)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_rows_and_wide_layers(gpu, dtype, m, n, k, group, zeros):
    """Prompts and batches: products are exact, so that a sum is off by its own roundings (at most three parts and 32 terms a product, the
    group's scale and the join: six sigma of as many as there are terms) and by the last one."""
    g = _g(m + n)
    x = torch.randn(m, k, generator=g).to(dtype)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((torch.rand(n, k // group, generator=g) + 0.5) / math.sqrt(k)).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    bias = torch.randn(n, generator=g).to(dtype)
    got = ops.linear_w4(ops.PackedW4(q.to(gpu), s.to(gpu), None if z is None else z.to(gpu), bias.to(gpu)), x.to(gpu))
    want, mag = O.linear_w4(x, q, s, z, bias)
    tol = u(dtype) * want.abs() * (1 + 2 * F) + 6 * math.sqrt(3 * k) * F * mag + 2 * F * (want.abs() + bias.double().abs()) + torch.finfo(dtype).tiny
    _within(got, want, tol, "rows")
