"""Outputs of the autoregressive-decoding operators that overlap what a call reads, or themselves: refused before any launch."""
import ctypes
import os
import subprocess

import pytest

from tts_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, Q = 4096, 1 << 20                                                   # never followed
ref = ctypes.byref


def _refused(fn, *args):
    L = _lib.lib()
    rc = getattr(L, "ttsamd_" + fn)(*args, None)
    assert rc == -1 and b"overlap" in L.ttsamd_last_error(), (fn, rc, L.ttsamd_last_error())


def _passes(fn, *args):
    """Past the checks: here, without a GPU, the launch itself fails (and on one this is not called)."""
    L = _lib.lib()
    rc = getattr(L, "ttsamd_" + fn)(*args, None)
    assert rc != -1, L.ttsamd_last_error()


def test_row_sets_against_brute_force(tmp_path):
    exe = str(tmp_path / "overlap")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests/native/overlap_driver.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and "overlap OK" in r.stdout, r.stdout + r.stderr


def test_rotary():
    plan = ops._RotaryPlan(P, 64, 0, 1.0)
    good = dict(x=Q, y=4 * Q, x_tstride=128, x_hstride=64, y_tstride=128, y_hstride=64, positions=P, position_bytes=8, tokens=4, heads=2, head_dim=64, dtype=0)
    R = lambda **kw: ref(ops._RotaryArgs(**{**good, **kw}))  # noqa: E731
    for kw in (dict(y_tstride=0), dict(y_hstride=0), dict(y_tstride=64), dict(y=Q + 4), dict(y=Q, y_tstride=256), dict(y=Q - 256), dict(x=Q, y=Q, x_hstride=0, y_hstride=0)):
        _refused("rotary", R(**kw), ref(plan))


def test_kv_append():
    cache = ref(ops._PagedKV(k=P, v=P, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, dtype=2, pages=4, kv_heads=4, page_size=16, head_dim=64))
    batch = ref(ops._PagedBatch(block_table=P, table_stride=4, seq_lens=P, q_starts=P, table_width=4, batch=2, max_new=1, max_len=64))
    es, row = 2, 12 * 64                                               # a fused projection: 4 query, 4 key, 4 value heads
    good = dict(q=Q, k=Q + 4 * 64 * es, v=Q + 8 * 64 * es, q_out=8 * Q, tokens=8, q_heads=4, qo_tstride=256, qo_hstride=64,
                **{n + s: v for n in "qkv" for s, v in (("_tstride", row), ("_hstride", 64))})
    A = lambda **kw: ref(ops._KvAppendArgs(**{**good, **kw}))  # noqa: E731
    for kw in (dict(qo_tstride=0), dict(qo_hstride=0), dict(q_out=good["k"], qo_tstride=row), dict(q_out=good["v"], qo_tstride=row), dict(q_out=Q, qo_tstride=256),
               dict(q_out=Q + 64 * es, qo_tstride=row), dict(q_out=good["k"] - 2, qo_tstride=row)):
        _refused("kv_append", A(**kw), cache, batch, None)


def test_paged_attention():
    cache = ref(ops._PagedKV(k=P, v=P, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, dtype=2, pages=4, kv_heads=4, page_size=16, head_dim=64))
    batch = ref(ops._PagedBatch(block_table=P, table_stride=4, seq_lens=P, q_starts=P, table_width=4, batch=2, max_new=1, max_len=64))
    good = dict(q=Q, out=4 * Q, q_tstride=256, q_hstride=64, o_tstride=256, o_hstride=64, tokens=8, q_heads=4, causal=1, window=0, scale=0.125)
    T = lambda **kw: ref(ops._PagedAttentionArgs(**{**good, **kw}))  # noqa: E731
    ws = (ctypes.c_void_p(P), ctypes.c_size_t(1 << 40))
    for kw in (dict(o_tstride=0), dict(o_hstride=0), dict(o_hstride=32), dict(out=Q + 128), dict(out=Q, o_tstride=512), dict(out=Q, o_tstride=64, o_hstride=512)):
        _refused("paged_attention", T(**kw), cache, batch, *ws)


def test_linear_w4():
    good = dict(x=Q, y=4 * Q, x_stride=128, y_stride=128, levels=P, scales=P, m=4, n=128, k=128, group=64, dtype=0, scale_dtype=1)
    W = lambda **kw: ref(ops._LinearW4Args(**{**good, **kw}))  # noqa: E731
    for kw in (dict(y=Q), dict(y_stride=0), dict(y_stride=100), dict(y=Q + 4), dict(y=Q + 3 * 512), dict(y=Q, m=1), dict(y=Q + 256, x_stride=256, y_stride=256)):
        _refused("linear_w4", W(**kw))


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the pointers here are not memory: only where nothing can be launched")
def test_what_lies_apart_is_not_refused():
    """Slices of one wider tensor side by side, and the same rows in place."""
    plan = ops._RotaryPlan(P, 64, 0, 1.0)
    R = dict(x=Q, y=Q + 512, x_tstride=256, x_hstride=64, y_tstride=256, y_hstride=64, positions=P, position_bytes=8, tokens=4, heads=2, head_dim=64, dtype=0)
    for kw in ({}, dict(y=Q), dict(y=Q + 256, x_hstride=128, y_hstride=128), dict(tokens=1, x_tstride=0, y_tstride=0), dict(y=4 * Q, x_hstride=0, x_tstride=0)):
        _passes("rotary", ref(ops._RotaryArgs(**{**R, **kw})), ref(plan))
    W = dict(x=Q, y=Q + 512, x_stride=256, y_stride=256, levels=P, scales=P, m=4, n=128, k=128, group=64, dtype=0, scale_dtype=1)
    for kw in ({}, dict(m=1, x_stride=0, y_stride=0), dict(x_stride=0, y=4 * Q)):
        _passes("linear_w4", ref(ops._LinearW4Args(**{**W, **kw})))
