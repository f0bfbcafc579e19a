"""fp32 attention on 16-bit products: what the smaller parts of an operand contribute, each by itself, and the error of the whole.

f = 2^-24.  x = x0 + x1 + x2: 8 bits each, so that a difference of two x from 2^-9 of them down is part 1's, from 2^-17 down part 2's."""
import math

import pytest
import torch

from tts_amd import ops

from .test_decode_gpu import F, Case, _g, _within

pytestmark = pytest.mark.gpu

# rows enough for the staged kernel, by widths and teams; and rows that stream
SHAPES = [(100, 130, 2, 4, 64), (257, 2000, 1, 1, 64), (200, 200, 1, 1, 64), (70, 90, 32, 64, 64), (64, 100, 1, 4, 96), (90, 700, 2, 4, 128), (100, 120, 1, 2, 192), (40, 60, 1, 2, 72), (9, 200, 1, 2, 128),
          (1, 300, 2, 2, 64), (1, 90, 1, 8, 104)]


def _case(gpu, shape):
    new, n, kv, heads, dim = shape
    c = Case(gpu, torch.float32, [new], [n], kv, heads, dim, 16, seed=n + dim)
    j = torch.arange(n)
    return c, c.table[0, j // 16].long().to(gpu), (j % 16).to(gpu)


# products whose large terms cancel exactly and leave one: q channels, key channels, what is left
d, e = 2.0 ** -10, 2.0 ** -19
LEFT = {"q1 k0": ([1 + d, 1], [1, -1], d), "q0 k1": ([1, -1], [1 + d, 1], d), "q2 k0": ([1 + e, 1], [1, -1], e), "q0 k2": ([1, -1], [1 + e, 1], e),
        "q1 k1": ([1 + d, 1, 1 + d, 1], [1 + d, -1 - d, -1, 1], d * d), "q12 k0": ([1 + d + e, 1 + d], [1, -1], e), "q0 k12": ([1, -1], [1 + d + e, 1 + d], e)}


@pytest.mark.parametrize("what", sorted(LEFT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_score_of_small_parts(gpu, shape, what):
    """Every third key has a score of 2 (all of it in the parts named), the others 0: sums of numbers that fp32 holds exactly.  What is off:
    p by 4 f (exponential), sums over n keys by 6 sqrt(n) f, the rest by 8 f, as in every fp32 test here."""
    q, k, left = LEFT[what]
    c, page, row = _case(gpu, shape)
    n, at = shape[1], [5 + 7 * i for i in range(len(q))]
    c.q.zero_()
    c.q[..., at] = torch.tensor(q, dtype=torch.float32)
    kk = torch.zeros(n, shape[2], shape[4])
    kk[::3, :, at] = torch.tensor(k, dtype=torch.float32)
    c.cache.k[page, :, row] = kk.to(gpu)
    assert float(torch.dot(torch.tensor(q, dtype=torch.float64), torch.tensor(k, dtype=torch.float64))) == left
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, scale=2.0 / left)
    want, mag, _ = c.want(2.0 / left)
    _within(got, want, (6 * math.sqrt(n) + 16) * F * mag + F * want.abs(), what)


@pytest.mark.parametrize("low,high", [(1, 1 << 7), (1 << 8, 1 << 15), (1, 1 << 22)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_of_small_parts(gpu, shape, low, high):
    """Scores of zero, and in every channel two values other than zero, 1 + m 2^-23 and -1: whatever order they are taken in, every sum of
    them or of their parts has 24 bits, and what is left is m 2^-23 / n, off by the division."""
    c, page, row = _case(gpu, shape)
    new, n, kv, heads, dim = shape
    g = _g(low + n)
    c.q.zero_()
    m = torch.randint(low, high, (kv, dim), generator=g)
    one = torch.randint(0, n, (kv, dim), generator=g)
    two = (one + torch.randint(1, n, (kv, dim), generator=g)) % n
    v = torch.zeros(n, kv, dim)
    v.scatter_(0, one[None], (1 + m.double() * 2.0 ** -23).float()[None])
    v.scatter_(0, two[None], torch.tensor(-1.0).expand(1, kv, dim))
    c.cache.v[page, :, row] = v.to(gpu)
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, causal=False)
    want = (m.double() * 2.0 ** -23 / n).repeat_interleave(heads // kv, 0)[None].expand(new, -1, -1)
    _within(got, want, 4 * F * want, "values")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_error_is_that_of_fp32(gpu, shape):
    """Root mean square against 64 bits: within three times that of the plain formula in fp32 on the CPU, both relative to sum p |v|."""
    c, page, row = _case(gpu, shape)
    new, n, kv, heads, dim = shape
    want, mag, _ = c.want(dim ** -0.5)
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch).cpu().double()
    k, v = (t[page, :, row].cpu().repeat_interleave(heads // kv, 1).transpose(0, 1) for t in (c.cache.k, c.cache.v))
    s = torch.matmul(c.q.transpose(0, 1), k.transpose(1, 2).contiguous()) * dim ** -0.5
    s = s.masked_fill(torch.arange(n)[None] > torch.arange(n - new, n)[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    plain = (torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)).transpose(0, 1)
    rms = lambda y: float((((y.double() - want) / mag) ** 2).mean().sqrt())  # noqa: E731
    assert rms(got) <= 3 * max(rms(plain), 0.3 * F), "%.3g, plain %.3g" % (rms(got), rms(plain))
