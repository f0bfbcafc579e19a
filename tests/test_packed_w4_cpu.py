"""The packed image of a 4-bit layer is a copy of everything that it was given, and what it takes is checked."""
import pytest
import torch

from tts_amd import _lib, ops


def _parts(n=40, k=128, group=32):
    g = torch.Generator().manual_seed(1)
    return (torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8), torch.rand(n, k // group, generator=g),
            torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8), torch.randn(n, generator=g))


def test_nothing_of_the_caller_is_kept():
    """Tiles in part and whole, so that padding copies and does not; written over, resized and freed afterwards."""
    for n in (40, 48):
        given = _parts(n)
        pw = ops.PackedW4(*given)
        kept = (pw.levels, pw.scales, pw.zeros, pw.bias)
        before = [t.clone() for t in kept]
        for t in given:
            t.zero_()
        assert all(torch.equal(a, b) for a, b in zip(kept, before))
        assert pw._pointers == tuple(t.data_ptr() for t in kept)
        assert not {t.untyped_storage().data_ptr() for t in kept} & {t.untyped_storage().data_ptr() for t in given}


def test_a_parameter_leaves_no_graph():
    q, s, z, b = _parts()
    pw = ops.PackedW4(q, torch.nn.Parameter(s), z, torch.nn.Parameter(b))
    assert not pw.scales.requires_grad and not pw.bias.requires_grad


def test_nbytes_is_the_images_size():
    q, s, z, b = _parts(40, 128, 32)
    tiles, chunks = 3, 1
    levels, groups = tiles * chunks * 256 * 4, tiles * 16 * 4
    assert ops.PackedW4(q, s).nbytes() == levels + 4 * groups
    assert ops.PackedW4(q, s, z, b).nbytes() == levels + 5 * groups + 4 * 40


def test_levels_of_other_ranks_are_refused():
    q, s, z, b = _parts()
    for bad in (q[0], q[..., None], q[None], torch.zeros((), dtype=torch.uint8)):
        with pytest.raises(_lib.TtsAmdError, match="qweight"):
            ops.PackedW4(bad, s)
