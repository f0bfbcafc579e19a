"""In-place calls of the autoregressive-decoding operators, and the outputs that they refuse."""
import pytest
import torch

from tts_amd import _lib, ops

from .test_decode_gpu import TYPES, Case, _g
from .test_decode_range_gpu import ROUTES

pytestmark = pytest.mark.gpu
E = _lib.TtsAmdError


@pytest.mark.parametrize("route", ROUTES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_over_its_own_queries(gpu, dtype, route):
    """The same bits in q's own rows, a slice of a wider tensor too, and where the rows are computed key by key."""
    new, n, kv, heads, dim = route
    c = Case(gpu, dtype, [new, 1], [n, 50], kv, heads, dim, 16, seed=n, trailing=2)
    for hidden in (False, True):
        if hidden:
            c.cache.v[int(c.table[0, (n - 1) // 16]), :, (n - 1) % 16, 0] = float("inf")
        q = c.q.to(gpu)
        want = ops.paged_attention(q, c.cache, c.batch)
        wide = torch.full((c.tokens, heads + 3, dim), 2.0, dtype=dtype, device=gpu)
        mine = wide[:, 1: heads + 1]
        mine.copy_(q)
        assert ops.paged_attention(mine, c.cache, c.batch, out=mine) is mine
        own = new + 1
        assert torch.equal(mine[:own].nan_to_num(3.0), want[:own].nan_to_num(3.0)) and torch.equal(mine[own:], q[own:])
        assert bool((wide[:, 0] == 2).all()) and bool((wide[:, heads + 1:] == 2).all())


def test_append_turns_the_queries_of_a_projection_in_place(gpu):
    dtype, kv, heads, dim = torch.bfloat16, 2, 4, 64
    c = Case(gpu, dtype, [20, 1], [40, 9], kv, heads, dim, 16, seed=1)
    fused = torch.randn(21, heads + 2 * kv, dim, generator=_g(3)).to(dtype).to(gpu)
    before = fused.clone()
    q, k, v = fused[:, :heads], fused[:, heads: heads + kv], fused[:, heads + kv:]
    plan = ops.Rotary(dim, device=gpu)
    want = ops.kv_append(c.cache, c.batch, k, v, rotary=plan, q=q)
    assert ops.kv_append(c.cache, c.batch, k, v, rotary=plan, q=q, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(fused[:, heads:], before[:, heads:])


def test_overlapping_outputs_are_refused(gpu):
    c = Case(gpu, torch.float32, [5], [20], 2, 4, 64, 16, seed=1)
    q = c.q.to(gpu)
    plan, pos = ops.Rotary(64, device=gpu), torch.arange(5, device=gpu)
    one = torch.zeros(1, 4, 64, device=gpu).expand(5, 4, 64)
    heads = torch.zeros(5, 1, 64, device=gpu).expand(5, 4, 64)
    longer = torch.zeros(6, 4, 64, device=gpu)
    longer[:5] = q
    for out in (one, heads):
        with pytest.raises(E, match="overlap"):
            ops.paged_attention(q, c.cache, c.batch, out=out)
        with pytest.raises(E, match="overlap"):
            ops.rotary(plan, q, pos, out=out)
        with pytest.raises(E, match="overlap"):
            ops.kv_append(c.cache, c.batch, q[:, :2], q[:, 2:], rotary=plan, q=q.clone(), q_out=out)
    for call in (lambda: ops.paged_attention(longer[:5], c.cache, c.batch, out=longer[1:]), lambda: ops.rotary(plan, longer[:5], pos, out=longer[1:]),
                 lambda: ops.kv_append(c.cache, c.batch, q[:, :2], q[:, 2:], rotary=plan, q=q.clone(), q_out=q)):
        with pytest.raises(E, match="overlap"):
            call()
    pw = ops.PackedW4.quantize(torch.randn(128, 128, device=gpu))
    x = torch.randn(4, 128, device=gpu)
    for out in (x, x[:1].expand(4, 128), torch.zeros(1, 128, device=gpu).expand(4, 128)):
        with pytest.raises(E, match="overlap"):
            ops.linear_w4(pw, x, out=out)
    wide = torch.zeros(4, 256, device=gpu)
    wide[:, :128] = x
    assert torch.equal(ops.linear_w4(pw, wide[:, :128], out=wide[:, 128:]), ops.linear_w4(pw, x))
    assert torch.equal(ops.linear_w4(pw, x[:1].expand(4, 128)), ops.linear_w4(pw, x[:1].repeat(4, 1)))      # an expanded input is fine
