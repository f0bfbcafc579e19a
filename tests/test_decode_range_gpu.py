"""Attention over a paged cache where scores are far from zero, or many keys weigh little: against closed forms and
oracle/decode.py.

u = half a step of the type, f = 2^-24, as in test_decode_gpu.py."""
import math

import pytest
import torch

from tts_amd import ops

from .test_decode_gpu import F, TYPES, Case, _g, _within, u

pytestmark = pytest.mark.gpu

# new tokens, keys, key heads, query heads, channels: one or two rows, streamed rows (one and two tiles), staged rows (one and two teams,
# all widths), each with the keys of a row whole and split over workgroups
ROUTES = [(1, 40, 1, 1, 64), (2, 70, 2, 2, 104), (1, 3000, 1, 2, 64), (1, 33, 2, 12, 80), (9, 60, 1, 3, 128), (20, 40, 2, 4, 64), (1, 2500, 1, 8, 192),
          (40, 90, 1, 1, 256), (130, 200, 2, 4, 64), (130, 150, 32, 64, 128), (100, 100, 1, 4, 96), (70, 1100, 1, 4, 128), (100, 130, 2, 4, 192), (110, 120, 1, 2, 256)]


def _at(c):
    """Pages and rows of the only sequence's keys, in order."""
    j = torch.arange(c.lens[0])
    return c.table[0, j // 16].long().to(c.gpu), (j % 16).to(c.gpu)


def _far(gpu, dtype, route, a, top, low):
    """Scores a * k0 with k0 = `top` for every seventh key and key 0, `low` for the others: the mean of the values of the former."""
    new, n, kv, heads, dim = route
    c = Case(gpu, dtype, [new], [n], kv, heads, dim, 16, seed=n + dim)
    c.q.zero_()
    c.q[..., 3] = a
    k = torch.zeros(n, kv, dim, dtype=torch.float64)
    k[..., 3] = low
    k[::7, :, 3] = top
    page, row = _at(c)
    c.cache.k[page, :, row] = k.to(dtype).to(gpu)
    return c


def _is_mean_of_the_top(c, got, dtype, what, rows=None, unlike=0.0):
    """Every p is 0 or the same: a sum of as many values as there are top keys, each in six partial products at most (fp32 in three
    parts), a rounding each, and the joins and the division.  unlike: how far p may differ between two parts of the keys: the mean moves by
    that share of one part's values and of itself."""
    n, new = c.lens[0], c.new[0]
    page, row = _at(c)
    v = c.cache.v[page, :, row].double().cpu()[::7].repeat_interleave(c.q.shape[1] // c.cache.kv_heads, 1)       # [top keys, heads, dim]
    count = torch.tensor([(n - new + i) // 7 + 1 for i in range(new)])
    want, mag = (torch.cumsum(x, 0)[count - 1] / count[:, None, None] for x in (v, v.abs()))
    tol = u(dtype) * want.abs() + (6 * count[:, None, None] + 40) * F * mag + 2 * unlike * mag + torch.finfo(dtype).tiny
    _within(got[:rows], want[:rows], tol[:rows], what)


@pytest.mark.parametrize("route", ROUTES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scores_far_from_zero(gpu, dtype, route):
    """Scores of some 2^36 of either sign, finite in every type: exact products, differences that leave p at 1 or 0."""
    for a, top, low in ((2.0 ** 15, 32000.0, 31744.0), (-2.0 ** 15, 31744.0, 32000.0), (2.0 ** 15, 5.0, -5.0), (1.0, 32000.0, -32000.0)):
        for scale in (64.0, 0.7 / 3, -64.0):
            c = _far(gpu, dtype, route, math.copysign(a, a * scale), top, low)
            _is_mean_of_the_top(c, ops.paged_attention(c.q.to(gpu), c.cache, c.batch, scale=scale), dtype, "%g %g %g %g" % (a, top, low, scale))
            # a value that only the last token sees: the others of its part of the keys row by row, where p is not rounded to 16 bits
            if route[0] > 1:
                c.cache.v[int(c.table[0, (route[1] - 1) // 16]), :, (route[1] - 1) % 16] = math.nan
                _is_mean_of_the_top(c, ops.paged_attention(c.q.to(gpu), c.cache, c.batch, scale=scale), dtype, "by the key", route[0] - 1,
                                    0.0 if dtype == torch.float32 else u(dtype))


@pytest.mark.parametrize("route", ROUTES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_scores_at_the_ends_of_the_range(gpu, dtype, route):
    """All scores of a row near -2^127 (or 2^127): no row that sees a key is empty."""
    big, less = 2.0 ** 63, 2.0 ** 63 * 1.984375
    for a, top, low, scale in ((-2.0 ** 63, big, less, 1.0), (-2.0 ** 63, big, big * 1.5, 1.25), (2.0 ** 63, less, big, 1.0), (2.0 ** 62, big, less, -1.5)):
        c = _far(gpu, dtype, route, a, top, low)
        _is_mean_of_the_top(c, ops.paged_attention(c.q.to(gpu), c.cache, c.batch, scale=scale), dtype, "%g %g %g" % (a, top, scale))


@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("new,n,kv,heads,dim", [(1, 4096, 1, 8, 64), (1, 9000, 2, 2, 128), (12, 4096, 1, 4, 192), (120, 5000, 1, 2, 64), (33, 4100, 8, 32, 128)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_light_keys_keep_their_weight(gpu, dtype, new, n, kv, heads, dim, where):
    """One key that outweighs each of the others by e^17.69 = 2^25.5, which only the others' values tell apart from nothing.

    A light key's p rounds to its type: u of itself, or half of the last place of a subnormal, 2^-25 where the heaviest key's is 2^11 at
    least (fp16): 2^-36 of the heaviest a key."""
    c = Case(gpu, dtype, [new], [n], kv, heads, dim, 16, seed=5)
    c.q.zero_()
    c.q[..., 1] = 8.0
    heavy = 0 if where == "first" else n - new
    page, row = _at(c)
    k, v = torch.zeros(n, kv, dim), torch.rand(n, kv, dim, generator=_g(2)) + 0.5
    k[..., 1] = -17.6875
    k[heavy], v[heavy] = 0, 0
    c.cache.k[page, :, row], c.cache.v[page, :, row] = k.to(dtype).to(gpu), v.to(dtype).to(gpu)
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, scale=0.125)
    want, mag, reach = c.want(0.125)
    delta = (6 * math.sqrt(dim) + 4) * F * reach
    rel = 2 * delta + 6 * math.sqrt(n) * F + (u(dtype) if dtype != torch.float32 else 0.0) + 8 * F
    lost = n * 2.0 ** -36 * 1.5 if dtype == torch.float16 else 0.0
    last = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2                       # half of the last place of a subnormal result
    assert float(want.abs().min()) > 5e-5
    _within(got, want, u(dtype) * want.abs() + rel * mag + lost + last, where)


@pytest.mark.parametrize("new,n,kv,heads,dim", [(1, 60, 2, 4, 64), (1, 1500, 1, 8, 128), (1, 700, 2, 6, 192), (9, 200, 1, 3, 80), (20, 300, 1, 4, 64), (16, 90, 2, 8, 128),
                                                (30, 400, 2, 4, 256), (1, 3000, 1, 2, 96)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_streamed_rows_keep_their_probabilities(gpu, dtype, new, n, kv, heads, dim):
    """Rows below the staged kernels' 96: a probability is a part of T and the remainder, rounded to T, u^2 of it off (and half of fp16's
    last step, 2^-36 of the heaviest key); nothing but the result is rounded to the type once."""
    c = Case(gpu, dtype, [new], [n], kv, heads, dim, 16, seed=dim)
    want, mag, reach = c.want(dim ** -0.5)
    delta = (6 * math.sqrt(dim) + 4) * F * reach
    rel = 2 * delta + 6 * math.sqrt(n) * F + 8 * F + u(dtype) ** 2
    lost = n * 2.0 ** -36 * float(c.cache.v[c.table[0].long()].nan_to_num(0, 0, 0).abs().max()) if dtype == torch.float16 else 0.0
    last = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    _within(ops.paged_attention(c.q.to(gpu), c.cache, c.batch), want, u(dtype) * want.abs() * (1 + rel) + rel * mag + lost + last, "two parts")
