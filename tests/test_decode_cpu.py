"""What the autoregressive-decoding operators refuse, how their indexes are bounded, and their plans: no GPU needed."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import pytest
import torch

from oracle import decode as O
from tts_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E = _lib.TtsAmdError
INVALID, UNSUPPORTED = -1, -2


def test_every_index_from_device_data_is_bounded(tmp_path):
    exe = str(tmp_path / "places")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests/native/places_driver.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and "places OK" in r.stdout, r.stdout + r.stderr


def test_structs_match_the_header(tmp_path):
    """Sizes and the offset of the last field of every argument struct, as a C compiler lays them out."""
    pairs = [("ttsamd_rotary_plan", ops._RotaryPlan), ("ttsamd_rotary_args", ops._RotaryArgs), ("ttsamd_paged_kv", ops._PagedKV),
             ("ttsamd_paged_batch", ops._PagedBatch), ("ttsamd_kv_append_args", ops._KvAppendArgs),
             ("ttsamd_paged_attention_args", ops._PagedAttentionArgs), ("ttsamd_linear_w4_args", ops._LinearW4Args)]
    src = '#include <stdio.h>\n#include "%s/include/tts_amd.h"\nint main(void) {\n' % ROOT
    for name, s in pairs:
        src += "".join('printf("%%zu ", offsetof(%s, %s));' % (name, f) for f, _ in s._fields_) + 'printf("%%zu\\n", sizeof(%s));\n' % name
    c = tmp_path / "s.c"
    c.write_text(src + "return 0; }\n")
    subprocess.run(["gcc", str(c), "-o", str(tmp_path / "s")], check=True)
    lines = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.strip().splitlines()
    for (name, s), line in zip(pairs, lines):
        assert [int(v) for v in line.split()] == [getattr(s, f).offset for f, _ in s._fields_] + [ctypes.sizeof(s)], name
    # the packed forms of the per-call structs are those mirrors' bytes
    for pack, s in ((ops._PACK_ROTARY, ops._RotaryArgs), (ops._PACK_APPEND, ops._KvAppendArgs), (ops._PACK_ATTENTION, ops._PagedAttentionArgs),
                    (ops._PACK_W4, ops._LinearW4Args)):
        values = [0.5 if t is ctypes.c_float else 1000 + i for i, (_, t) in enumerate(s._fields_)]
        assert pack(*values) == bytes(s(*values)), s


@pytest.mark.parametrize("rd,kw", [(64, {}), (32, {"scaling": {"kind": "linear", "factor": 4.0}}), (128, {"scaling": {"kind": "base", "factor": 8.0}}),
                                   (64, {"scaling": {"kind": "ramp", "factor": 8.0, "trained_len": 4096}}), (2, {"base": 500000.0})])
def test_rotary_plan_keeps_far_positions(rd, kw):
    """turns * position modulo 2^64 is the angle itself: against the frequency in exact fractions, at positions up to 2^31."""
    plan = ops.Rotary(128, rd, device="cpu", **kw)
    base, sc = kw.get("base", 10000.0), kw.get("scaling", {"kind": "none"})
    if sc["kind"] == "base":
        base = base * 8.0 ** (rd / (rd - 2.0))
    freq = [base ** (-2.0 * i / rd) for i in range(rd // 2)]
    if sc["kind"] == "linear":
        freq = [f / 4.0 for f in freq]
    if sc["kind"] == "ramp":
        keep = [min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / 31.0)) for f in freq]
        freq = [f / 8.0 * (1 - k) + f * k for f, k in zip(freq, keep)]
        assert abs(plan.amplitude - (0.1 * math.log(8.0) + 1.0)) < 1e-7
    circle = Fraction(62831853071795864769252867665590057683943, 10 ** 40)
    for f, t in zip(freq, plan.turns.tolist()):
        for p in (1, 1000, 1234567, 2 ** 31 - 1, -77):
            got, want = Fraction((t * p) % 2 ** 64, 2 ** 64), (Fraction(f) * p / circle) % 1
            d = abs(got - want)
            assert min(d, 1 - d) < abs(p) * Fraction(1, 2 ** 64), (f, p)


def test_python_refusals():
    f = torch.float32
    R = ops.Rotary(64, device="cpu")
    for bad in (dict(rotary_dim=3), dict(rotary_dim=66), dict(scaling={"kind": "other"}), dict(scaling={"kind": "linear", "factor": 0.0}),
                dict(scaling={"kind": "linear", "factor": 2.0, "low": 1}), dict(rotary_dim=2, scaling={"kind": "base", "factor": 2.0}),
                dict(inv_freq=[1.0]), dict(inv_freq=[math.inf] * 32), dict(inv_freq=[1.0] * 32, scaling={"kind": "linear", "factor": 2.0})):
        with pytest.raises(E):
            ops.Rotary(64, device="cpu", **bad)
    x, pos = torch.zeros(4, 2, 64), torch.arange(4)
    for a in ((R, x.double(), pos), (R, x[0], pos), (R, torch.zeros(4, 2, 32), pos), (R, x, pos[:3]), (R, x, pos.float()),
              (R, torch.zeros(4, 64, 2).transpose(1, 2), pos), (R, x, torch.arange(8)[::2]), (R, x, pos)):      # the last: not on the GPU
        with pytest.raises(E):
            ops.rotary(*a)
    K = lambda *s, t=f: torch.zeros(s, dtype=t)  # noqa: E731
    for k, v in ((K(2, 2, 16, 64), K(2, 2, 16, 32)), (K(2, 2, 16), K(2, 2, 16)), (K(2, 2, 16, 60), K(2, 2, 16, 60)), (K(2, 2, 16, 264), K(2, 2, 16, 264)),
                 (K(2, 2, 16, 64), K(2, 2, 16, 64, t=torch.float16)), (K(2, 2, 16, 64, t=torch.float64), K(2, 2, 16, 64, t=torch.float64)),
                 (K(0, 2, 16, 64), K(0, 2, 16, 64)), (K(2, 2, 16, 65)[..., 1:], K(2, 2, 16, 65)[..., 1:]), (K(2, 2, 64, 16).transpose(2, 3),) * 2):
        with pytest.raises(E):
            ops.PagedKV(k, v)
    i = torch.int32
    T, L, S = torch.zeros(3, 4, dtype=i), torch.zeros(3, dtype=i), torch.zeros(4, dtype=i)
    for a in ((T.long(), L, S, 1), (T, L.long(), S, 1), (T, L, S[:3], 1), (T[:2], L, S, 1), (T.t(), L, S, 1), (T, L, S, -1), (T, L, S, 1, -1),
              (torch.zeros(4, 3, dtype=i).t(), L, S, 1), (torch.zeros(70000, 0, dtype=i), torch.zeros(70000, dtype=i), torch.zeros(70001, dtype=i), 1)):
        with pytest.raises(E):
            ops.PagedBatch(*a)
    cache, batch = ops.PagedKV(K(2, 2, 16, 64), K(2, 2, 16, 64)), ops.PagedBatch(T, L, S, 1)
    k = K(5, 2, 64)
    for a, kw in (((k, k[:4]), {}), ((k, K(5, 2, 32)), {}), ((k.half(), k.half()), {}), ((k, k), dict(q=K(4, 2, 64))), ((k, k), dict(q=K(5, 2, 32))),
                  ((k, k), dict(positions=torch.arange(5))), ((k, k), dict(rotary=ops.Rotary(32, device="cpu"))), ((k, k), dict(q_out=k)),
                  ((k, k), dict(rotary=R, positions=torch.arange(4))), ((k, k), {})):
        with pytest.raises(E):
            ops.kv_append(cache, batch, *a, **kw)
    for q, kw in ((K(5, 3, 64), {}), (K(5, 4, 32), {}), (K(5, 4, 64).half(), {}), (K(5, 4), {}), (K(5, 4, 64), dict(window=-1)), (K(5, 4, 64), {})):
        with pytest.raises(E):
            ops.paged_attention(q, cache, batch, **kw)
    w, s = torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 2)
    for a in ((w.int(), s), (w, s.double()), (w, torch.zeros(8, 3)), (w, torch.zeros(8, 8)), (w, torch.zeros(7, 2)), (w, s, torch.zeros(8, 2)),
              (w, s, torch.zeros(8, 1, dtype=torch.uint8)), (w, s, None, torch.zeros(7)), (w, torch.zeros(8, 0))):
        with pytest.raises(E):
            ops.PackedW4(*a)
    pw = ops.PackedW4(w, s, bias=torch.zeros(8))
    for x in (torch.zeros(2, 64), torch.zeros(2, 128).double(), torch.zeros(2, 128).half(), torch.zeros(128, 2).t(), torch.zeros(128), torch.zeros(2, 128)):
        with pytest.raises(E):
            ops.linear_w4(pw, x)


def _refused(fn, want, *args):
    L = _lib.lib()
    rc = getattr(L, "ttsamd_" + fn)(*args, None)
    assert rc == want, (fn, rc, L.ttsamd_last_error())
    assert fn.split("_")[0].encode() in L.ttsamd_last_error()


def test_c_refusals_come_before_any_launch():
    """The C entries check what the kernels assume; the pointers here are never followed."""
    for what, arguments in (("rotary", 1), ("kv_append", 3), ("paged_attention", 4), ("linear_w4", 0)):
        ops._entry(what, arguments)                                         # what the Python views call leaves the library's own attribute alone
    ref, P = ctypes.byref, 4096
    plan = ops._RotaryPlan(P, 64, 0, 1.0)
    good = dict(x=P, y=P, x_tstride=64, x_hstride=64, y_tstride=64, y_hstride=64, positions=P, position_bytes=8, tokens=1, heads=1, head_dim=64, dtype=0)
    R = lambda **kw: ref(ops._RotaryArgs(**{**good, **kw}))  # noqa: E731
    for kw in (dict(dtype=3), dict(x=None), dict(positions=None), dict(position_bytes=2), dict(head_dim=62), dict(tokens=-1), dict(heads=-1)):
        _refused("rotary", INVALID, R(**kw), ref(plan))
    _refused("rotary", INVALID, R(), ref(ops._RotaryPlan(P, 63, 0, 1.0)))
    _refused("rotary", INVALID, R(), ref(ops._RotaryPlan(None, 64, 0, 1.0)))
    _refused("rotary", INVALID, None, ref(plan))
    _refused("rotary", UNSUPPORTED, R(heads=1 << 20), ref(plan))
    assert _lib.lib().ttsamd_rotary(R(tokens=0, x=None), ref(plan), None) == 0
    kv = dict(k=P, v=P, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, dtype=2, pages=4, kv_heads=4, page_size=16, head_dim=64)
    C = lambda **kw: ref(ops._PagedKV(**{**kv, **kw}))  # noqa: E731
    bt = dict(block_table=P, table_stride=4, seq_lens=P, q_starts=P, table_width=4, batch=2, max_new=1, max_len=64)
    B = lambda **kw: ref(ops._PagedBatch(**{**bt, **kw}))  # noqa: E731
    ap = dict(k=P, v=P, k_tstride=256, k_hstride=64, v_tstride=256, v_hstride=64, tokens=2)
    A = lambda **kw: ref(ops._KvAppendArgs(**{**ap, **kw}))  # noqa: E731
    at = dict(q=P, out=P, q_tstride=256, q_hstride=64, o_tstride=256, o_hstride=64, tokens=2, q_heads=4, causal=1, window=0, scale=0.125)
    T = lambda **kw: ref(ops._PagedAttentionArgs(**{**at, **kw}))  # noqa: E731
    ws = (ctypes.c_void_p(P), ctypes.c_size_t(1 << 40))
    bad_kv = [dict(k=None), dict(dtype=9), dict(pages=0), dict(kv_heads=0), dict(page_size=0), dict(head_dim=0), dict(k=P + 8), dict(v_row=60), dict(k_page=-8)]
    bad_bt = [dict(seq_lens=None), dict(q_starts=None), dict(block_table=None), dict(batch=-1), dict(batch=65536), dict(table_width=-1),
              dict(max_new=-1), dict(max_len=-1), dict(table_stride=-1)]
    for kw in bad_kv:
        _refused("kv_append", INVALID, A(), C(**kw), B(), None)
        _refused("paged_attention", INVALID, T(), C(**kw), B(), *ws)
    for kw in bad_bt:
        _refused("kv_append", INVALID, A(), C(), B(**kw), None)
        _refused("paged_attention", INVALID, T(), C(), B(**kw), *ws)
    for dim in (12, 264):
        _refused("kv_append", UNSUPPORTED, A(), C(head_dim=dim), B(), None)
        _refused("paged_attention", UNSUPPORTED, T(), C(head_dim=dim), B(), *ws)
    for kw in (dict(k=None), dict(tokens=-1), dict(q=P, q_heads=4), dict(q=P, q_out=P, q_heads=0), dict(positions=P, position_bytes=3)):
        _refused("kv_append", INVALID, A(**kw), C(), B(), None)
    _refused("kv_append", INVALID, A(), C(), B(), ref(ops._RotaryPlan(P, 66, 0, 1.0)))
    for kw in (dict(q=None), dict(out=None), dict(q=P + 4), dict(q_tstride=250), dict(o_hstride=4), dict(q_heads=0), dict(q_heads=6), dict(window=-1),
               dict(tokens=-1)):
        _refused("paged_attention", INVALID, T(**kw), C(), B(), *ws)
    assert _lib.lib().ttsamd_paged_attention(T(tokens=0), C(), B(), *ws, None) == 0
    w4 = dict(x=P, y=P, x_stride=128, y_stride=16, levels=P, scales=P, zeros=None, bias=None, m=1, n=16, k=128, group=64, dtype=0, scale_dtype=1)
    W = lambda **kw: ref(ops._LinearW4Args(**{**w4, **kw}))  # noqa: E731
    for kw in (dict(x=None), dict(levels=None), dict(scales=None), dict(dtype=4), dict(scale_dtype=-1), dict(m=-1), dict(k=0), dict(k=96), dict(levels=P + 4)):
        _refused("linear_w4", INVALID, W(**kw))
    _refused("linear_w4", UNSUPPORTED, W(group=16))
    assert _lib.lib().ttsamd_linear_w4(W(m=0, x=None), None) == 0


def test_w4_image_holds_every_level_in_its_place():
    g = torch.Generator().manual_seed(3)
    n, k, group = 21, 160, 32
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s, z = torch.rand(n, k // group, generator=g), torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    pw = ops.PackedW4(q, s, z)
    assert tuple(pw.levels.shape) == (2, 2, 4, 16, 4) and tuple(pw.scales.shape) == (2, 8, 16) and tuple(pw.zeros.shape) == (2, 8, 16)
    level = lambda i, j: (int(q[i, j // 2]) >> (4 * (j % 2))) & 15  # noqa: E731
    for i in range(32):
        for j in range(256):
            word = int(pw.levels[i // 16, j // 128, j % 32 // 8, i % 16, j % 128 // 32]) & 0xFFFFFFFF
            assert (word >> (4 * (j % 8 // 2) + 16 * (j % 2))) & 15 == (level(i, j) if i < n and j < k else 0)
            if j % group == 0:
                inside = i < n and j < k
                assert float(pw.scales[i // 16, j // group, i % 16]) == (float(s[i, j // group]) if inside else 0.0)
                assert int(pw.zeros[i // 16, j // group, i % 16]) == (int(z[i, j // group]) if inside else 0)


def test_w4_image_is_its_own():
    """One group of one chunk: the image's scales and zeros have the order of the given ones, but no memory in common with them."""
    scales, zeros = torch.rand(33, 1)[1:], torch.full((33, 1), 3, dtype=torch.uint8)[1:]
    pw = ops.PackedW4(torch.zeros(32, 64, dtype=torch.uint8), scales, zeros)
    before = pw.scales.clone()
    scales.zero_(), zeros.zero_()
    assert torch.equal(pw.scales, before) and bool((pw.zeros == 3).all())
    assert pw.scales.data_ptr() % 16 == 0 and pw.zeros.data_ptr() % 16 == 0


def test_oracle_against_plain_softmax():
    """The 64-bit oracle itself, on a batch whose pages lie in order: torch's own softmax."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(4, 2, 8, 16, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(3, 4, 16, generator=g, dtype=torch.float64)
    out, _, _ = O.attend(q, k, v, [[2, 0, 3]], [19], [0, 3], 0.25)
    kk, vv = (torch.cat([c[2], c[0], c[3]], 1)[:, :19] for c in (k, v))
    for h in range(4):
        s = q[:, h] @ kk[h // 2].T * 0.25
        s = s.masked_fill(torch.arange(19)[None] > torch.arange(16, 19)[:, None], -math.inf)
        assert torch.allclose(out[:, h], torch.softmax(s, -1) @ vv[h // 2], atol=1e-12)
