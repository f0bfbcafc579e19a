"""GPU parity of the autoregressive-decoding operators (rotary positions, the append to a paged cache, attention over it, 4-bit
products) against oracle/decode.py in 64 bits.

Tolerances.  u = half a step of the type (finfo.eps / 2), f = 2^-24.  A result rounds once: u |y|.  Before that
  rotary   the angle is off by at most 1.6 f, the Taylor sums by 1.5 f, the factor and the two products by 2 f: 8 f A (|x1| + |x2|)
  attend   a score is a sum of d products in fp32, off by 6 sqrt(d) f (six sigma of as many roundings) of sum |q k| scale, plus 4 f of it
           for the scale and the exponential's argument: delta; p is off by delta up and down the softmax: 2 delta, plus 6 sqrt(n) f for
           its sums over n keys, plus u where p itself is rounded to the 16-bit type: all of it times sum p |v|
  w4       products are exact but for the level offset of at most 31 in 24 bits: 6 sqrt(k) f of 8 sum |x w|  (an offset level is at most
           31 against a mean |level - zero| of about 4)"""
import math

import pytest
import torch

from oracle import decode as O
from tts_amd import _lib, ops

pytestmark = pytest.mark.gpu
F = 2.0 ** -24
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def u(dtype):
    return torch.finfo(dtype).eps / 2


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, tol, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    assert not bool(bad.any()), "%s: %d values off, worst %.3g over its bound (value %.6g, wanted %.6g)" % (
        what, int(bad.sum()), float((off - tol)[bad].max()), float(got[bad][0]), float(want[bad][0]))


# ---------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,heads,dim,rd,inter,scaling", [
    (1, 1, 2, 2, False, None), (3, 5, 64, 64, False, None), (7, 3, 80, 40, True, {"kind": "linear", "factor": 4.0}),
    (33, 2, 98, 34, False, {"kind": "base", "factor": 8.0}), (5, 16, 128, 0, False, None), (1000, 9, 48, 48, True, None),
    (2, 4, 256, 128, False, {"kind": "ramp", "factor": 8.0, "trained_len": 4096}), (700, 32, 128, 128, False, None)])
def test_rotary(gpu, dtype, tokens, heads, dim, rd, inter, scaling):
    g = _g(tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    pos = torch.randint(-5, 3_000_000, (tokens,), generator=g)
    plan = ops.Rotary(dim, rd, interleaved=inter, scaling=scaling, device=gpu)
    rope = [10000.0 ** (-2.0 * i / rd) for i in range(rd // 2)]
    amp = 1.0
    if scaling and scaling["kind"] == "linear":
        rope = [f / 4.0 for f in rope]
    elif scaling and scaling["kind"] == "base":
        rope = [(10000.0 * 8.0 ** (rd / (rd - 2.0))) ** (-2.0 * i / rd) for i in range(rd // 2)]
    elif scaling:
        keep = [min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / 31.0)) for f in rope]
        rope, amp = [f / 8.0 * (1 - k) + f * k for f, k in zip(rope, keep)], 0.1 * math.log(8.0) + 1.0
    want = O.turned(x, pos, rope, amp, inter)
    mag = O.turned(x, torch.zeros_like(pos), rope, amp, inter).abs()
    pair = mag.clone()
    if rd:
        one, two = (slice(0, rd, 2), slice(1, rd, 2)) if inter else (slice(0, rd // 2), slice(rd // 2, rd))
        pair[..., one] = pair[..., two] = mag[..., one] + mag[..., two]
    # 2.3e-10: a position of 3e6 times a frequency rounded in 53 bits, in radians
    tol = u(dtype) * want.abs() * (1 + 8 * F) + pair * (8 * F + 1e-9) + torch.finfo(dtype).tiny
    got = ops.rotary(plan, x.to(gpu), pos.to(gpu))
    _within(got, want, tol, "rotary")
    assert torch.equal(got[..., rd:].cpu(), x[..., rd:])
    # in place, int32 positions: the same bits
    y = x.to(gpu).clone()
    assert ops.rotary(plan, y, pos.to(gpu).int(), out=y) is y and torch.equal(y, got)
    # strided, unaligned rows in and out: the same bits
    wide = torch.zeros(tokens, heads + 1, dim + 3, dtype=dtype, device=gpu)
    wide[:, 1:, 1: dim + 1] = x.to(gpu)
    out = torch.full((tokens, heads, dim + 5), 7.0, dtype=dtype, device=gpu)
    ops.rotary(plan, wide[:, 1:, 1: dim + 1], pos.to(gpu), out=out[..., 3: dim + 3])
    assert torch.equal(out[..., 3: dim + 3], got) and bool((out[..., :3] == 7).all()) and bool((out[..., dim + 3:] == 7).all())


def test_rotary_gradient_is_the_inverse_turn(gpu):
    """<rotary(x), w> has the gradient rotary(w, inverse): against autograd of the plain formula, and against differences."""
    g = _g(5)
    x, w = (torch.randn(6, 3, 32, generator=g) for _ in range(2))
    pos = torch.randint(0, 5000, (6,), generator=g)
    plan = ops.Rotary(32, 16, interleaved=True, device=gpu)
    freq = [10000.0 ** (-2.0 * i / 16) for i in range(8)]
    leaf = x.double().requires_grad_()
    a = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64)
    x1, x2 = leaf[..., 0:16:2], leaf[..., 1:16:2]
    y = torch.cat([torch.stack([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1).flatten(-2), leaf[..., 16:]], -1)
    (y * w.double()).sum().backward()
    got = ops.rotary(plan, w.to(gpu), pos.to(gpu), inverse=True)
    _within(got, leaf.grad, 8 * F * (w.double().abs().amax() * 2 + leaf.grad.abs()), "gradient")
    # differences: the map is linear, so a step of any size is exact but for rounding
    d = torch.randn(6, 3, 32, generator=g)
    f = lambda t: (ops.rotary(plan, t.to(gpu), pos.to(gpu)).double().cpu() * w.double()).sum()  # noqa: E731
    slope = float(f(x + d) - f(x - d)) / 2
    n = x.numel()
    assert abs(slope - float((got.double().cpu() * d.double()).sum())) <= 64 * F * math.sqrt(n) * float(d.abs().max() + x.abs().max()) * float(w.abs().max())


# ------------------------------------------------------------------------------------------------------------ the cache
class Case:
    """Sequences with pages dealt out at random from a pool; what no sequence owns holds NaN and infinities."""

    def __init__(self, gpu, dtype, new, lens, kv_heads, heads, dim, page, seed=0, trailing=0, table_extra=0, far_pages=0):
        g = _g(seed)
        self.new, self.lens, self.dtype, self.page, self.gpu = list(new), list(lens), dtype, page, gpu
        owned = [-(-max(c, 0) // page) for c in lens]
        pages = sum(owned) + 2 + far_pages
        order = torch.randperm(pages, generator=g)
        width = max(owned + [0]) + table_extra
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        self.k, self.v = (torch.randn(pages, kv_heads, page, dim, generator=g).to(dtype) for _ in range(2))
        trash = torch.tensor([math.nan, math.inf, -math.inf])
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, c in enumerate(lens):
            for i in range(owned[b]):
                self.table[b, i] = order[at]
                used[order[at], : min(page, c - i * page)] = True
                at += 1
        for c in (self.k, self.v):
            junk = trash[torch.randint(0, 3, c.shape, generator=g)].to(dtype)
            c.copy_(torch.where(used[:, None, :, None], c, junk))
        self.starts = torch.tensor([0] + list(torch.tensor(self.new).cumsum(0)), dtype=torch.int32)
        self.tokens = sum(self.new) + trailing
        self.q = torch.randn(self.tokens, heads, dim, generator=g).to(dtype)
        self.cache = ops.PagedKV(self.k.to(gpu), self.v.to(gpu))
        self.batch = ops.PagedBatch(self.table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), self.starts.to(gpu), max(self.new + [0]),
                                    max(lens + [0]))

    def want(self, scale, causal=True, window=0):
        return O.attend(self.q, self.cache.k.cpu(), self.cache.v.cpu(), self.table.tolist(), self.lens, self.starts.tolist(), scale, causal, window)

    def check(self, got, scale=None, causal=True, window=0, what=""):
        dim = self.q.shape[2]
        scale = dim ** -0.5 if scale is None else scale
        want, mag, reach = self.want(scale, causal, window)
        delta = (6 * math.sqrt(dim) + 4) * F * reach
        rel = 2 * delta + 6 * math.sqrt(max(self.lens + [1])) * F + (u(self.dtype) if self.dtype != torch.float32 else 0.0) + 8 * F
        mine = ~torch.isnan(want).all(-1).all(-1)
        _within(got[mine.to(got.device)], want[mine], u(self.dtype) * want[mine].abs() + rel * mag[mine] + torch.finfo(self.dtype).tiny, what)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lens,kv,heads,dim,page,rd,inter", [
    ([1], [1], 1, 1, 8, 1, 8, False), ([1, 1, 1], [17, 16, 1], 2, 4, 64, 16, 64, False), ([5, 0, 3], [5, 9, 40], 1, 3, 40, 7, 20, True),
    ([130, 1, 77], [130, 300, 90], 4, 4, 128, 32, 64, False), ([300], [300], 8, 16, 256, 64, 0, False)])
def test_kv_append(gpu, dtype, new, lens, kv, heads, dim, page, rd, inter):
    c = Case(gpu, dtype, new, lens, kv, heads, dim, page, seed=dim + page, trailing=2)
    g = _g(9)
    k, v = (torch.randn(c.tokens, kv, dim, generator=g).to(dtype) for _ in range(2))
    plan = ops.Rotary(dim, rd, interleaved=inter, device=gpu)
    before_k, before_v = c.cache.k.cpu().clone(), c.cache.v.cpu().clone()
    q = ops.kv_append(c.cache, c.batch, k.to(gpu), v.to(gpu), rotary=plan, q=c.q.to(gpu))
    got_k, got_v = c.cache.k.cpu(), c.cache.v.cpu()
    own = sum(new)
    pos = torch.cat([torch.arange(n - a, n) for a, n in zip(new, lens)])
    # the rotation is rotary()'s own, bit for bit (itself held to 64 bits above)
    want_k = ops.rotary(plan, k[:own].to(gpu), pos.to(gpu)).cpu()
    assert torch.equal(q[:own].cpu(), ops.rotary(plan, c.q[:own].to(gpu), pos.to(gpu)).cpu())
    at = 0
    for b, (start, n, where, slots) in enumerate(O.places(c.table.tolist(), lens, c.starts.tolist(), page, c.k.shape[0], c.tokens)):
        for i in range(n):
            pg, row = slots[where[i]]
            before_k[pg, :, row], before_v[pg, :, row] = want_k[start + i], v[start + i]
            at += 1
    assert at == own
    same = lambda a, b: torch.equal(a.view(torch.int16 if dtype != torch.float32 else torch.int32), b.view(torch.int16 if dtype != torch.float32 else torch.int32))  # noqa: E731,E501
    assert same(got_k, before_k) and same(got_v, before_v)          # every other row of the cache as it was, NaN and all
    # without a plan nothing turns; positions of the caller's own
    ops.kv_append(c.cache, c.batch, k.to(gpu), v.to(gpu))
    where = [s[p] for _, n, w, s in O.places(c.table.tolist(), lens, c.starts.tolist(), page, c.k.shape[0], c.tokens) for p in w]
    assert all(torch.equal(c.cache.k.cpu()[pg, :, r], k[i]) for i, (pg, r) in enumerate(where))
    other = torch.arange(c.tokens) * 3 - 4
    ops.kv_append(c.cache, c.batch, k.to(gpu), v.to(gpu), rotary=plan, positions=other.to(gpu))
    turned = ops.rotary(plan, k.to(gpu), other.to(gpu)).cpu()
    assert all(torch.equal(c.cache.k.cpu()[pg, :, r], turned[i]) for i, (pg, r) in enumerate(where))


def test_kv_append_takes_no_write_outside_the_pages(gpu):
    """Pages that are not there, positions before the first and behind the table: those tokens write nothing; the others all do."""
    new, lens = [4, 3, 2], [2, 12, 9]                                # sequence 0: two tokens at positions -2, -1
    c = Case(gpu, torch.float32, new, lens, 2, 2, 16, 4, seed=3)
    c.table[1, 2] = c.k.shape[0] + 5                                 # positions 8..11 of sequence 1: no such page
    table = c.table[:, :2].contiguous().to(gpu)                      # sequence 2's position 8 is behind the table
    c.table[1, 2] = -7
    for t, page1 in ((table, -1), (c.table.to(gpu), -7)):
        cache = ops.PagedKV.allocate(c.k.shape[0], 4, 2, 16, device=gpu)
        batch = ops.PagedBatch(t, c.batch.seq_lens, c.batch.q_starts, 4)
        k = torch.randn(9, 2, 16, generator=_g(1)).to(gpu)
        ops.kv_append(cache, batch, k, -k)
        want = torch.zeros_like(cache.k)
        for start, n, pos, where in O.places(t.tolist(), lens, c.starts.tolist(), 4, c.k.shape[0], 9):
            for i, p in enumerate(pos):
                if p >= 0 and where[p] is not None:
                    want[where[p][0], :, where[p][1]] = k[start + i]
        assert torch.equal(cache.k, want) and torch.equal(cache.v, -want)


# --------------------------------------------------------------------------------------------------------- attention
ATTEND = [
    # new, lens, kv_heads, heads, dim, page: single tokens
    ([1], [1], 1, 1, 8, 1), ([1], [2], 1, 1, 64, 16), ([1, 1, 1, 1], [63, 64, 65, 1], 2, 2, 64, 16), ([1, 1], [0, 5], 2, 4, 64, 4),
    ([1, 1], [1000, 777], 2, 6, 128, 64), ([1], [5000], 1, 8, 64, 32), ([1, 1, 0, 1], [129, 31, 40, 256], 1, 16, 80, 24),
    ([1], [700], 2, 34, 96, 16), ([2, 1, 0], [90, 513, 4], 2, 2, 64, 16), ([1, 1], [33, 700], 2, 4, 128, 5), ([2], [1030], 1, 1, 40, 16),
    ([1, 1], [2600, 90], 1, 2, 104, 16), ([3, 1], [40, 41], 1, 1, 64, 16), ([1, 1], [300, 50], 1, 1, 256, 128), ([1], [513], 3, 3, 40, 7),
    # chunks
    ([2], [2], 1, 1, 64, 16), ([17, 1, 33], [17, 40, 33], 2, 2, 64, 16), ([5, 64], [100, 64], 1, 3, 128, 1), ([70], [333], 2, 4, 72, 24),
    ([129, 128, 127], [129, 200, 500], 1, 2, 128, 64), ([40], [40], 1, 8, 256, 16), ([300], [310], 2, 2, 32, 13), ([9, 6], [4, 6], 1, 2, 64, 8),
    # chunks with enough rows to be staged for 128 at a time: whole and part tiles, all widths of a head
    ([129, 64, 1, 33, 70], [129, 190, 400, 33, 65], 16, 16, 64, 16), ([40, 90], [40, 350], 16, 64, 128, 64), ([33, 34], [97, 40], 16, 64, 80, 1),
    ([70, 10], [77, 300], 16, 32, 256, 24), ([65, 100], [500, 99], 32, 32, 40, 32), ([128, 128], [256, 129], 16, 32, 200, 8),
    ([129, 1, 70], [129, 400, 65], 2, 8, 64, 16), ([300], [300], 1, 1, 128, 13), ([260, 5], [300, 5], 1, 1, 256, 16),
    # more of them than the chip holds at once, by one and by two teams of waves
    ([100, 97, 3], [300, 100, 50], 32, 64, 64, 16), ([130, 70, 5], [130, 200, 40], 64, 64, 64, 24), ([130, 70, 5], [130, 200, 40], 64, 64, 128, 16),
    # the same with the keys split over workgroups
    ([70, 3], [1100, 700], 1, 4, 128, 64), ([300], [900], 1, 1, 256, 24), ([90, 20], [640, 33], 2, 6, 80, 1), ([65, 64], [600, 64], 1, 4, 200, 8),
    ([257], [2000], 1, 1, 64, 16), ([1], [3000], 1, 2, 64, 16), ([9], [2500], 1, 3, 128, 8), ([40], [1500], 1, 1, 256, 32)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lens,kv,heads,dim,page", ATTEND)
def test_paged_attention(gpu, dtype, new, lens, kv, heads, dim, page):
    c = Case(gpu, dtype, new, lens, kv, heads, dim, page, seed=sum(lens) + dim, trailing=3, table_extra=1)
    out = torch.full(c.q.shape, 5.0, dtype=dtype, device=gpu)
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, out=out)
    assert got is out and bool((out[sum(new):] == 5).all())           # behind the last sequence: as it was
    c.check(got, what="causal")
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, window=max(1, max(lens) // 3), scale=0.3)
    c.check(got, scale=0.3, window=max(1, max(lens) // 3), what="window")


# heads between the widths that are powers of two, whole and in part
BETWEEN = [
    ([1, 1], [700, 33], 2, 4, 16), ([1], [3000], 1, 8, 32), ([9, 0, 2], [100, 40, 2], 1, 3, 1), ([129, 64, 1], [129, 190, 400], 2, 4, 16),
    ([70, 90], [70, 350], 16, 64, 24), ([300], [1200], 1, 1, 13), ([130, 70, 5], [130, 200, 40], 64, 64, 16)]


@pytest.mark.parametrize("dim", [88, 96, 136, 192])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lens,kv,heads,page", BETWEEN)
def test_paged_attention_heads_between_the_widths(gpu, dtype, dim, new, lens, kv, heads, page):
    c = Case(gpu, dtype, new, lens, kv, heads, dim, page, seed=sum(lens) + dim, trailing=2)
    c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch), what="causal")
    c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch, window=60, scale=-0.1), scale=-0.1, window=60, what="window")


@pytest.mark.parametrize("dim,heads", [(96, 2), (192, 2), (192, 1)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_attention_non_finite_values_between_the_widths(gpu, dtype, dim, heads):
    """An infinity and a NaN that only the last tokens of a chunk see."""
    new, n = 80, 200
    c = Case(gpu, dtype, [new], [n], 1, heads, dim, 8, seed=3)
    for j, value in ((n - 10, math.inf), (n - 6, math.nan)):
        c.cache.v[int(c.table[0, j // 8]), :, j % 8, dim - 1] = value
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch).cpu()
    want, _, _ = c.want(dim ** -0.5, True, 0)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)) and bool(torch.isfinite(want[: new - 10]).all())
    assert not bool(torch.isfinite(got[new - 10:, :, dim - 1]).any())
    sub = got[: new - 10].double() - want[: new - 10]
    assert float(sub.abs().max()) < 40 * u(dtype) + 1e-5


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lens,window,kv", [([1, 1], [200, 33], 0, 2), ([40, 3], [200, 33], 0, 2), ([40, 90], [200, 90], 50, 2), ([1], [90], 1, 2),
                                                ([140, 65], [200, 90], 50, 2), ([170], [840], 0, 2)])
def test_paged_attention_not_causal(gpu, dtype, new, lens, window, kv):
    c = Case(gpu, dtype, new, lens, kv, 2 * kv, 64, 16, seed=7)
    c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch, causal=False, window=window), causal=False, window=window)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,kv", [(1, 2), (20, 2), (150, 2), (150, 1)])
def test_paged_attention_bad_pages_and_sizes_hold_no_key(gpu, dtype, new, kv):
    """Pages outside the pool, a table narrower than the lengths, starts beyond the tokens: what is there is attended, nothing faults."""
    c = Case(gpu, dtype, [new, new], [160, 170], kv, 4, 64, 16, seed=new)
    for col, page in ((0, -3), (3, 10 ** 6), (9, 2 ** 31 - 1)):
        c.table[0, col] = page
    c.table = c.table[:, :10].contiguous()                            # sequence 1 reaches position 169: its last keys have no column
    c.batch = ops.PagedBatch(c.table.to(gpu), c.batch.seq_lens, c.batch.q_starts, new)
    c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch), what="pages")
    c.table[1, :] = -1                                                # a sequence with no page at all: zeros
    c.batch = ops.PagedBatch(c.table.to(gpu), c.batch.seq_lens, c.batch.q_starts, new)
    got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch)
    assert bool((got[new:] == 0).all())
    c.check(got, what="no page")
    c.starts = torch.tensor([-4, new + 3, 10 ** 9], dtype=torch.int32)
    c.batch = ops.PagedBatch(c.table.to(gpu), c.batch.seq_lens, c.starts.to(gpu), new)
    c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch), what="starts")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kv", [2, 1])
def test_paged_attention_computes_more_than_it_was_sized_for(gpu, dtype, kv):
    c = Case(gpu, dtype, [70, 1, 200], [90, 400, 250], kv, 4, 64, 16, seed=2)
    for most in ((1, 1), (0, 0), (7, 40), (65, 100)):
        c.batch = ops.PagedBatch(c.table.to(gpu), c.batch.seq_lens, c.batch.q_starts, max_new=most[0], max_len=most[1])
        c.check(ops.paged_attention(c.q.to(gpu), c.cache, c.batch), what=str(most))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,kv,scale", [(1, 2, None), (90, 2, None), (70, 1, None), (70, 1, -0.2), (70, 1, 0.0), (1, 2, -0.2), (1, 2, 0.0)])
def test_paged_attention_strides_and_large_scores(gpu, dtype, new, kv, scale):
    """A layer's slice of a cache of many layers, q as a slice of one projection, out in a wider tensor; scores in the hundreds; scales that
    are negative or zero."""
    heads = 4
    c = Case(gpu, dtype, [new, new], [300, 120], kv, heads, 64, 16, seed=4)
    pages = c.k.shape[0]
    pool = torch.full((pages, 3, 2, 16, kv, 64), math.nan, dtype=dtype, device=gpu)   # [pages, layers, k/v, rows, heads, dim]
    pool[:, 1, 0], pool[:, 1, 1] = c.k.to(gpu).transpose(1, 2), c.v.to(gpu).transpose(1, 2)
    cache = ops.PagedKV(pool[:, 1, 0].transpose(1, 2), pool[:, 1, 1].transpose(1, 2))
    fused = torch.randn(c.tokens, heads + 4, 64, generator=_g(1)).to(dtype).to(gpu)
    mine = fused[:, 2: heads + 2]
    mine.copy_((c.q * 20).to(gpu))
    wide = torch.full((c.tokens, heads + 2, 64), 3.0, dtype=dtype, device=gpu)
    ops.paged_attention(mine, cache, c.batch, scale=scale, out=wide[:, 1: heads + 1])
    assert bool((wide[:, 0] == 3).all()) and bool((wide[:, heads + 1] == 3).all())
    c.q = mine.cpu()
    c.check(wide[:, 1: heads + 1], scale=scale, what="strided")


@pytest.mark.parametrize("kv,heads,n", [(1, 2, 180), (2, 8, 180), (1, 4, 900), (1, 1, 900)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_attention_non_finite_values_reach_only_who_sees_them(gpu, dtype, kv, heads, n):
    """NaN and infinities in keys or values of tokens that a row does not see (later ones of its chunk, those out of its window) take no
    part in it."""
    new = 100
    c = Case(gpu, dtype, [new], [n], kv, heads, 64, 16, seed=8)
    for j, value in ((n - 60, math.nan), (n - 30, math.inf), (n - 9, -math.inf)):
        page, row = int(c.table[0, j // 16]), j % 16
        (c.cache.k if j == n - 30 else c.cache.v)[page, :, row, 5] = value
    for window in (0, 20):
        got = ops.paged_attention(c.q.to(gpu), c.cache, c.batch, window=window)
        want, _, _ = c.want(64 ** -0.5, True, window)
        assert torch.equal(torch.isfinite(got).cpu(), torch.isfinite(want)), window
        fine = [i for i in range(new) if bool(torch.isfinite(want[i]).all())]
        assert len(fine) >= 40
        sub = got[fine].double().cpu() - want[fine]
        assert float(sub.abs().max()) < 40 * u(dtype) + 1e-5


def test_paged_attention_positions_beyond_32_bits_of_bytes(gpu):
    """A pool whose pages lie further apart than 2^31 elements."""
    dtype = torch.bfloat16
    c = Case(gpu, dtype, [1, 30], [100, 70], 1, 2, 64, 16, seed=6)
    pages = c.k.shape[0]
    stride = (1 << 31) // (pages - 3) // 8 * 8 + 8
    pool = torch.empty((pages - 1) * stride + 2 * 16 * 64, dtype=dtype, device=gpu)
    k = pool.as_strided((pages, 1, 16, 64), (stride, 1024, 64, 1))
    v = pool[1024:].as_strided((pages, 1, 16, 64), (stride, 1024, 64, 1))
    k.copy_(c.k.to(gpu)), v.copy_(c.v.to(gpu))
    assert (pages - 1) * stride * 2 > 1 << 32
    cache = ops.PagedKV(k, v)
    c.check(ops.paged_attention(c.q.to(gpu), cache, c.batch))
    new_k = torch.randn(31, 1, 64, generator=_g(3)).to(dtype).to(gpu)
    ops.kv_append(cache, c.batch, new_k, new_k)
    c.cache = ops.PagedKV(k.contiguous(), v.contiguous())
    c.check(ops.paged_attention(c.q.to(gpu), cache, c.batch))
    assert torch.equal(cache.k[int(c.table[0, 6]), :, 3], new_k[0])


@pytest.mark.parametrize("trailing", [0, 500, 9000])
def test_paged_attention_workspace_stays_small_when_tokens_are_padding(gpu, trailing):
    """A long cache read by one token of a call sized for thousands: few or no parts, the same result."""
    import ctypes

    c = Case(gpu, torch.bfloat16, [1, 1], [4000, 3500], 2, 16, 64, 16, seed=13, trailing=trailing)
    a = ops._PagedAttentionArgs(tokens=c.tokens, q_heads=16, causal=1, scale=1.0)
    need = _lib.lib().ttsamd_paged_attention_workspace_bytes(bytes(a), ctypes.c_void_p(c.cache._ref), ctypes.c_void_p(c.batch._ref))
    assert need <= 256 << 20 and (trailing > 0 or need > 0)
    out = torch.full(c.q.shape, 2.0, dtype=c.dtype, device=gpu)
    ops.paged_attention(c.q.to(gpu), c.cache, c.batch, out=out)
    assert bool((out[2:] == 2).all())
    c.check(out, what="padded")


# ------------------------------------------------------------------------------------------------------------------- w4
def _w4(dtype, m, n, k, group, zeros, bias, seed):
    g = _g(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((torch.rand(n, k // group, generator=g) + 0.5) / math.sqrt(k)).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return x, q, s, z, b


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k,group,zeros,bias", [
    (1, 1, 32, 32, False, False), (1, 16, 128, 128, True, True), (2, 100, 256, 64, False, True), (5, 17, 96, 32, True, False),
    (1, 1024, 1024, 64, False, True), (16, 33, 640, 128, True, True), (17, 64, 320, 64, False, False), (33, 250, 1056, 32, True, True),
    (64, 48, 512, 128, False, True), (100, 20, 192, 64, True, False), (1, 40, 8192, 128, False, True), (4, 4096, 64, 64, True, True),
    (260, 70, 384, 128, False, False),
    # few and many rows where a workgroup has two and four tiles of outputs, the last of them in part
    (3, 8200, 96, 32, True, True), (5, 8199, 192, 64, False, True), (6, 8195, 160, 32, True, False), (16, 8200, 384, 128, True, True),
    (1, 16400, 128, 64, True, False), (4, 16390, 640, 128, False, True), (2, 16386, 64, 32, False, False), (20, 8203, 320, 64, True, True)])
def test_linear_w4(gpu, dtype, m, n, k, group, zeros, bias):
    x, q, s, z, b = _w4(dtype, m, n, k, group, zeros, bias, m + n + k)
    want, mag = O.linear_w4(x, q, s, z, b)
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    pw = ops.PackedW4(up(q), up(s), up(z), up(b))
    tol = u(dtype) * want.abs() + 8 * 6 * math.sqrt(k) * F * mag + 2 * F * want.abs() + torch.finfo(dtype).tiny
    if b is not None:
        tol = tol + 2 * F * b.double().abs()
    got = ops.linear_w4(pw, x.to(gpu))
    _within(got, want, tol, "w4")
    # rows of a wider x into rows of a wider y
    wide = torch.full((m, k + 8), 9.0, dtype=dtype, device=gpu)
    wide[:, 3: k + 3] = x.to(gpu)
    out = torch.full((m, n + 5), 4.0, dtype=dtype, device=gpu)
    ops.linear_w4(pw, wide[:, 3: k + 3], out=out[:, 2: n + 2])
    assert torch.equal(out[:, 2: n + 2], got) and bool((out[:, :2] == 4).all()) and bool((out[:, n + 2:] == 4).all())


@pytest.mark.parametrize("scale_dtype", TYPES, ids=str)
def test_linear_w4_scales_of_any_type_and_non_finite_rows(gpu, scale_dtype):
    x, q, s, z, _ = _w4(torch.float32, 3, 30, 256, 64, True, False, 1)
    x[1, 70] = math.nan
    x[2, 255] = math.inf
    pw = ops.PackedW4(q.to(gpu), s.to(scale_dtype).to(gpu), z.to(gpu))
    want, mag = O.linear_w4(x[:1], q, s.to(scale_dtype), z)
    got = ops.linear_w4(pw, x.to(gpu))
    _within(got[:1], want, 8 * 6 * 16 * F * mag, "scales")            # a row is its own: NaN and infinity next to it change nothing
    assert bool(torch.isnan(got[1]).all()) and not bool(torch.isfinite(got[2]).any())


@pytest.mark.parametrize("dtype,m,n,k,group", [(torch.float32, 5, 50, 384, 128), (torch.float16, 17, 33, 256, 64), (torch.bfloat16, 3, 16, 96, 32)])
def test_linear_w4_infinities_and_the_largest_values(gpu, dtype, m, n, k, group):
    """An infinity takes every output to the infinity (or NaN, at a weight of zero) that the plain sum gives; a finite sum of the type's
    largest values stays finite."""
    x, q, s, z, _ = _w4(dtype, m, n, k, group, True, False, 4)
    s = s.sign() * 2.0 ** -8
    x[0, k // 3], x[1, 5], x[1, k - 1], x[2, 0] = math.inf, -math.inf, -math.inf, torch.finfo(dtype).max
    level = torch.stack([q & 15, q >> 4], -1).view(n, k).double()
    w = (level - z.repeat_interleave(group, 1).double()) * s.repeat_interleave(group, 1).double()
    want = (x.double()[:, None] * w).sum(-1)
    assert not bool(torch.isfinite(want[:2]).any()) and bool(torch.isfinite(want[2:]).all())
    got = ops.linear_w4(ops.PackedW4(q.to(gpu), s.to(gpu), z.to(gpu)), x.to(gpu)).cpu().double()
    assert torch.equal(torch.isnan(got[:2]), torch.isnan(want[:2]))
    same = ~torch.isnan(want[:2])
    assert torch.equal(got[:2][same], want[:2][same])
    # k roundings of sums no larger than the sum of the products' sizes (six times it where x (16 + q) meets x (16 + z)), one to the type
    mag = (x.double()[2:, None] * w).abs().sum(-1)
    assert bool(((got[2:] - want[2:]).abs() <= 6 * k * F * mag + torch.finfo(dtype).eps / 2 * want[2:].abs()).all())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_is_within_half_a_step(gpu, group, zeros):
    w = torch.randn(40, 256, generator=_g(2)).to(gpu)
    pw = ops.PackedW4.quantize(w, group, zeros=zeros)
    back = ops.linear_w4(pw, torch.eye(256, device=gpu)).t()
    f = w.view(40, -1, group)
    step = (f.amax(-1).clamp(min=0) - f.amin(-1).clamp(max=0)) / 15 if zeros else f.abs().amax(-1) / 7.5
    # half a step inside the range; with a zero point rounded to a level another half at the ends
    assert bool(((back - w).abs().view(40, -1, group) <= (1.01 if zeros else 0.51) * step[..., None] + 1e-6).all())


# ----------------------------------------------------------------------------------------------- together, captured, at once
class Layer:
    """A decoder layer's attention half: 4-bit products in, append with rotation, attention, 4-bit product out."""

    def __init__(self, gpu, dtype, kv, heads, dim, width, seed):
        g = _g(seed)
        self.kv, self.heads, self.dim = kv, heads, dim
        self.raw = []
        for n, k in (((heads + 2 * kv) * dim, width), (width, heads * dim)):
            q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
            s = ((torch.rand(n, k // 64, generator=g) + 0.5) * (0.25 / math.sqrt(k))).to(dtype)
            self.raw.append((q, s, None, torch.randn(n, generator=g).to(dtype)))
        self.w_in, self.w_out = (ops.PackedW4(*(None if t is None else t.to(gpu) for t in r)) for r in self.raw)
        self.plan = ops.Rotary(dim, device=gpu)

    def __call__(self, x, cache, batch):
        fused = ops.linear_w4(self.w_in, x).view(x.shape[0], self.heads + 2 * self.kv, self.dim)
        q, k, v = fused[:, : self.heads], fused[:, self.heads: self.heads + self.kv], fused[:, self.heads + self.kv:]
        q = ops.kv_append(cache, batch, k, v, rotary=self.plan, q=q)
        o = ops.paged_attention(q, cache, batch)
        return fused, q, o, ops.linear_w4(self.w_out, o.view(x.shape[0], -1))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_layer_reads_prompts_and_makes_tokens(gpu, dtype):
    """Ragged prompts in one chunk, then single tokens of all requests: every stage against 64 bits on that stage's own inputs."""
    kv, heads, dim, width, page = 2, 4, 64, 256, 16
    layer = Layer(gpu, dtype, kv, heads, dim, width, 3)
    prompts, steps = [70, 1, 33], 3
    table = torch.randperm(24, generator=_g(5)).view(3, 8).to(torch.int32)
    cache = ops.PagedKV.allocate(24, page, kv, dim, dtype, gpu)
    lens = [0, 0, 0]
    freq = [10000.0 ** (-2.0 * i / dim) for i in range(dim // 2)]
    for step in range(1 + steps):
        new = prompts if step == 0 else [1, 1, 1]
        before = list(lens)
        lens = [a + b for a, b in zip(lens, new)]
        starts = [0, new[0], new[0] + new[1], sum(new)]
        x = torch.randn(sum(new), width, generator=_g(100 + step)).to(dtype)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
        batch = ops.PagedBatch(table.to(gpu), i32(lens), i32(starts), max(new), max(lens))
        fused, q, o, y = layer(x.to(gpu), cache, batch)
        for (w, s, z, b), inp, out in ((layer.raw[0], x, fused.view(sum(new), -1)), (layer.raw[1], o.cpu().view(sum(new), -1), y)):
            want, mag = O.linear_w4(inp, w, s, z, b)
            _within(out, want, (u(dtype) + 2 * F) * want.abs() + 8 * 6 * math.sqrt(inp.shape[1]) * F * mag + 2 * F * b.double().abs(), "product")
        pos = torch.cat([torch.arange(a, b) for a, b in zip(before, lens)])
        f = fused.cpu()
        for got, src in ((q, f[:, :heads]), (None, f[:, heads: heads + kv])):
            want = O.turned(src, pos, freq)
            if got is None:
                at = [(int(table[b, p // page]), p % page) for b in range(3) for p in range(before[b], lens[b])]
                got = torch.stack([cache.k[pg, :, r] for pg, r in at])
                assert torch.equal(torch.stack([cache.v[pg, :, r] for pg, r in at]).cpu(), f[:, heads + kv:])
            half = dim // 2
            size = src.double().abs()
            pair = torch.cat([size[..., :half] + size[..., half:]] * 2, -1)
            _within(got, want, u(dtype) * want.abs() * (1 + 8 * F) + pair * 8 * F, "turned")
        want, mag, reach = O.attend(q.cpu(), cache.k.cpu(), cache.v.cpu(), table.tolist(), lens, starts, dim ** -0.5)
        rel = 2 * (6 * math.sqrt(dim) + 4) * F * reach + 6 * math.sqrt(max(lens)) * F + (u(dtype) if dtype != torch.float32 else 0.0) + 8 * F
        _within(o, want, u(dtype) * want.abs() + rel * mag, "attention")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,room", [(1, 64), (1, 640), (80, 100)])
def test_captured_steps_follow_what_is_written_into_the_batch(gpu, dtype, new, room):
    """A layer captured once and replayed with other lengths, starts and pages, eager work between: each replay the bits of the eager call."""
    kv, heads, dim, width, page, seqs = 2, 8, 64, 128, 16, 3
    layer = Layer(gpu, dtype, kv, heads, dim, width, 7)
    columns = -(-room // page)
    pages = seqs * columns
    fixed = dict(table=torch.zeros(seqs, columns, dtype=torch.int32, device=gpu), lens=torch.zeros(seqs, dtype=torch.int32, device=gpu),
                 starts=torch.zeros(seqs + 1, dtype=torch.int32, device=gpu), x=torch.zeros(seqs * new, width, dtype=dtype, device=gpu))
    caches = [ops.PagedKV.allocate(pages, page, kv, dim, dtype, gpu) for _ in range(2)]
    batch = ops.PagedBatch(fixed["table"], fixed["lens"], fixed["starts"], new, room)

    def write(k):
        g = _g(40 + k)
        n = [new, max(1, new // (k + 1)), new if k % 2 else 1]
        start = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32)
        lens = torch.tensor([min(room, n[i] + 7 * k + (room * i) // 3) for i in range(3)], dtype=torch.int32)
        fixed["table"].copy_(torch.randperm(pages, generator=g).view(seqs, columns).int())
        fixed["lens"].copy_(lens), fixed["starts"].copy_(start)
        fixed["x"].copy_(torch.randn(seqs * new, width, generator=g).to(dtype))
        k0, v0 = (torch.randn(caches[0].k.shape, generator=g).to(dtype) for _ in range(2))
        for c in caches:
            c.k.copy_(k0), c.v.copy_(v0)
        return sum(n)

    write(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(fixed["x"], caches[0], batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(fixed["x"], caches[0], batch)
    for k in range(5):
        own = write(k)
        graph.replay()
        want = layer(fixed["x"], caches[1], batch)
        torch.cuda.synchronize()
        for a, b in zip(out[:3], want[:3]):
            assert torch.equal(a[:own], b[:own]), k
        assert torch.equal(out[3][:own], want[3][:own]) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_two_threads_on_two_streams(gpu):
    """The same plan, cache pages and batch objects used by two threads at once, each on its own stream."""
    import threading

    c = Case(gpu, torch.bfloat16, [1] * 4, [1500, 900, 1200, 64], 2, 8, 64, 16, seed=11)
    q = c.q.to(gpu)
    want = ops.paged_attention(q, c.cache, c.batch)
    plan = ops.Rotary(64, device=gpu)
    turned = ops.rotary(plan, q, torch.arange(4, device=gpu))
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                a, b = ops.paged_attention(q, c.cache, c.batch), ops.rotary(plan, q, torch.arange(4, device=gpu))
                s.synchronize()
                if not (torch.equal(a, want) and torch.equal(b, turned)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_empty_calls(gpu):
    """No tokens, no sequences, no rows: nothing is launched, results have their shape."""
    cache = ops.PagedKV.allocate(2, 4, 1, 8, device=gpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    none = ops.PagedBatch(torch.zeros(0, 3, dtype=torch.int32, device=gpu), i32(), i32(0), 0)
    some = ops.PagedBatch(i32(0, 1).view(1, 2), i32(3), i32(0, 0), 1)
    flat = ops.PagedBatch(torch.zeros(1, 0, dtype=torch.int32, device=gpu), i32(3), i32(0, 2), 2)
    x = torch.ones(0, 1, 8, device=gpu)
    for b in (none, some):
        assert ops.paged_attention(x, cache, b).shape == (0, 1, 8)
        ops.kv_append(cache, b, x, x)
    two = torch.ones(2, 1, 8, device=gpu)
    ops.kv_append(cache, flat, two, two)                              # a table without columns: no place to write, no key to read
    assert bool((ops.paged_attention(two, cache, flat) == 0).all()) and bool((cache.k == 0).all())
    out = torch.full((2, 1, 8), 3.0, device=gpu)
    assert bool((ops.paged_attention(two, cache, some, out=out) == 3).all())
    assert ops.rotary(ops.Rotary(8, device=gpu), x, torch.zeros(0, dtype=torch.int64, device=gpu)).shape == (0, 1, 8)
    pw = ops.PackedW4.quantize(torch.randn(4, 64, device=gpu))
    assert ops.linear_w4(pw, torch.ones(0, 64, device=gpu)).shape == (0, 4)
