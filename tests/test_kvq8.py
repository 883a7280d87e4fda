"""CPU tests of the paged 8-bit cache: byte layout and bounds of the shared header (a host
build), the rotation's frequencies, and every refusal of the entry points, which happens
before anything touches the GPU."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest
import torch

import kvq8_ref as R
from hipgpt_amd import _lib, kvcache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # any aligned non-null value: checks fail before any dereference


def test_layout_and_bounds_on_the_host(tmp_path):
    exe = str(tmp_path / "kvq8_bounds")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-D__HIP_PLATFORM_AMD__",
                    "-I" + os.path.join(ROOT, "include"), "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "cpp", "kvq8_bounds.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("ps,D", [(32, 32), (64, 128), (128, 64)])
def test_reference_layout_is_the_headers(ps, D):
    """kvq8_ref's byte order, spelled out from the header's words."""
    at = R.v_bytes(ps, D)
    assert sorted(at.reshape(-1)) == list(range(ps * D))
    for t in (0, 5, 17, 31, ps - 1):
        for d in (0, 1, 15, 16, 31, D - 1):
            i3, i0, i4 = t % 32 // 16, t % 16 // 4, t % 4
            i2, i1 = d % 32 // 16, d % 16
            want = ((((t // 32 * (D // 32) + d // 32) * 4 + i0) * 16 + i1) * 2 + i2) * 8 + i3 * 4 + i4
            assert at[t, d] == want
    c = np.random.default_rng(1).integers(-127, 128, (3, 2, ps, D))
    k, v = R.pool_to_codes(*R.codes_to_pool(c))
    assert np.array_equal(k, c) and np.array_equal(v, c)


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (26, 1.0)])
def test_rope_freqs(rot, base):
    f = kvcache.rope_freqs(rot, base, device="cpu").numpy()
    want = np.array([base ** (-2.0 * i / rot) / (2 * math.pi) for i in range(rot // 2)])
    # the fixed point is off by half its last place, 2^-65 of a turn, whatever the number
    # (2^-65 / 3.9e-7 = 7e-14 of the smallest here); both sides round in 64 bits on the way
    assert (np.abs(f.astype(np.float64) / 2.0**64 - want) <= 2.0**-65 + 8 * 2.0**-53 * want).all()
    # a position times the fixed-point number keeps the fraction of a turn exactly
    pos = 1048573
    exact = Fraction(int(f[0]) * pos % 2**64, 2**64)
    assert abs(float(exact) - (want[0] * pos) % 1.0) <= pos * want[0] * 2.0**-52


def test_rope_freqs_refusals():
    L = _lib.lib()
    f = (ctypes.c_uint64 * 8)()
    for args in ((None, 8, 1e4), (f, 0, 1e4), (f, 7, 1e4), (f, 8, 0.5), (f, 8, float("nan")), (f, 8, float("inf"))):
        assert L.hipgpt_rope_freqs(*args) == _lib.ERR_INVALID
    with pytest.raises(_lib.HipgptError):
        kvcache.rope_freqs(6, 0.0, device="cpu")


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, page_stride=2 * 64 * 64, head_stride=64 * 64, scale_page_stride=2,
             scale_head_stride=1, num_pages=4, page_size=64, heads=2, head_dim=64)
    d.update(kw)
    return ctypes.byref(_lib.KvQ8Cache(**d))


def batch(**kw):
    d = dict(block_table=P, table_stride=4, lens=P, cu_new=P, batch=2, max_pages=4, max_new=5)
    d.update(kw)
    return ctypes.byref(_lib.KvQ8Batch(**d))


def calls(c, b, T):
    """The four entry points on otherwise good arguments."""
    L = _lib.lib()
    s = (128, 64)
    yield L.hipgpt_kvq8_append(c, b, T, P, P, P, P, 2, *s, *s, *s, *s, P, 64, 0, 0, 0, None)
    yield L.hipgpt_kvq8_read(c, b, T, P, P, *s, *s, 0, None)
    yield L.hipgpt_attn_prefill_kvq8(c, b, T, P, P, 2, *s, *s, -1.0, 0, 0, 1, None, 0, None)


BAD_CACHES = [
    (dict(k=0), "INVALID"), (dict(v=0), "INVALID"), (dict(k_scale=0), "INVALID"), (dict(v_scale=0), "INVALID"),
    (dict(num_pages=0), "INVALID"), (dict(heads=-1), "INVALID"), (dict(page_size=0), "INVALID"),
    (dict(head_dim=0), "INVALID"), (dict(page_size=48), "UNSUPPORTED"), (dict(page_size=16), "UNSUPPORTED"),
    (dict(page_size=256), "UNSUPPORTED"), (dict(head_dim=48), "UNSUPPORTED"), (dict(head_dim=512), "UNSUPPORTED"),
    (dict(head_stride=64 * 64 - 16), "INVALID"), (dict(page_stride=0), "INVALID"), (dict(scale_page_stride=0), "INVALID"),
    (dict(scale_head_stride=0), "INVALID"), (dict(k=P + 8), "UNSUPPORTED"), (dict(v=P + 4), "UNSUPPORTED"),
    (dict(page_stride=3 * 64 * 64, head_stride=64 * 64 + 8), "UNSUPPORTED"),
    (dict(page_stride=2 * 64 * 64 + 4), "UNSUPPORTED"),
    # heads and pages that overlap
    (dict(page_stride=64 * 64), "INVALID"), (dict(page_stride=2 * 64 * 64, head_stride=64 * 64 + 16), "INVALID"),
    (dict(page_stride=64 * 64, head_stride=3 * 64 * 64), "INVALID"), (dict(scale_page_stride=1), "INVALID"),
    (dict(page_stride=1 << 62, head_stride=1 << 62), "INVALID"),
]
BAD_BATCHES = [
    (dict(block_table=0), 7), (dict(lens=0), 7), (dict(batch=0), 7), (dict(max_pages=0), 7), (dict(max_new=0), 7),
    (dict(table_stride=-1), 7), (dict(table_stride=0), 7), (dict(table_stride=3), 7), (dict(), 0), (dict(), -3),
    (dict(cu_new=0, max_new=5), 2), (dict(cu_new=0, max_new=1), 3),
]


@pytest.mark.parametrize("kw,why", BAD_CACHES)
def test_bad_caches_are_refused(kw, why):
    want = getattr(_lib, "ERR_" + why)
    c = cache(**kw)
    if "heads" in kw:
        assert list(calls(c, batch(), 7)) == [want] * 3
    else:
        assert all(rc == want for rc in calls(c, batch(), 7))


@pytest.mark.parametrize("kw,T", BAD_BATCHES)
def test_bad_batches_are_refused(kw, T):
    assert all(rc == _lib.ERR_INVALID for rc in calls(cache(), batch(**kw), T))
    L = _lib.lib()
    assert L.hipgpt_kvq8_read(None, batch(), 7, P, P, 128, 64, 128, 64, 0, None) == _lib.ERR_INVALID
    assert L.hipgpt_kvq8_read(cache(), None, 7, P, P, 128, 64, 128, 64, 0, None) == _lib.ERR_INVALID


def test_append_refusals():
    f = _lib.lib().hipgpt_kvq8_append
    s = (128, 64)

    def call(q=P, q_out=P, k=P, v=P, Hq=2, qs=s, qo=s, ks=s, vs=s, freqs=P, rot=64, dt=0):
        return f(cache(), batch(), 7, q, q_out, k, v, Hq, *qs, *qo, *ks, *vs, freqs, rot, 0, dt, 0, None)

    for kw in (dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(Hq=0), dict(dt=2), dict(dt=-1),
               dict(rot=0), dict(rot=-2), dict(rot=63), dict(rot=66)):
        assert call(**kw) == _lib.ERR_INVALID, kw
    for kw in (dict(q=P + 4), dict(q_out=P + 8), dict(k=P + 2), dict(v=P + 4), dict(qs=(130, 64)), dict(qo=(128, 66)),
               dict(ks=(128, 62)), dict(vs=(127, 64)), dict(ks=(132, 64), dt=1)):
        assert call(**kw) == _lib.ERR_UNSUPPORTED, kw


def test_read_refusals():
    f = _lib.lib().hipgpt_kvq8_read
    assert f(cache(), batch(), 7, None, P, 128, 64, 128, 64, 0, None) == _lib.ERR_INVALID
    assert f(cache(), batch(), 7, P, None, 128, 64, 128, 64, 0, None) == _lib.ERR_INVALID
    assert f(cache(), batch(), 7, P, P, 128, 64, 128, 64, 9, None) == _lib.ERR_INVALID
    assert f(cache(), batch(), 7, P, P, 126, 64, 128, 64, 0, None) == _lib.ERR_UNSUPPORTED
    assert f(cache(), batch(), 7, P, P + 8, 128, 64, 128, 64, 0, None) == _lib.ERR_UNSUPPORTED


def test_attention_refusals():
    L = _lib.lib()
    s = (128, 64)

    def both(q=P, o=P, Hq=4, qs=s, os_=s, scale=-1.0, dt=0, odt=0, c=None):
        c = c or cache()
        pre = L.hipgpt_attn_prefill_kvq8(c, batch(), 7, q, o, Hq, *qs, *os_, scale, dt, odt, 1, None, 0, None)
        dec = L.hipgpt_attn_decode_kvq8(c, batch(cu_new=0, max_new=1), q, o, Hq, *qs, *os_, scale, dt, odt, 1, None, 0,
                                        None)
        assert pre == dec
        return pre

    for kw in (dict(q=None), dict(o=None), dict(Hq=0), dict(Hq=3), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(dt=2), dict(odt=-1)):
        assert both(**kw) == _lib.ERR_INVALID, kw
    huge = batch(max_new=1 << 30)
    assert L.hipgpt_attn_prefill_kvq8(cache(), huge, 1 << 30, P, P, 4, *s, *s, -1.0, 0, 0, 1, None, 0,
                                      None) == _lib.ERR_UNSUPPORTED
    for kw in (dict(odt=1), dict(q=P + 4), dict(o=P + 8), dict(qs=(126, 64)), dict(os_=(128, 63)),
               dict(dt=1, odt=1, qs=(132, 64)), dict(c=cache(head_dim=48))):
        assert both(**kw) == _lib.ERR_UNSUPPORTED, kw
    # decode: one row per sequence, and a workspace for several splits
    dec = L.hipgpt_attn_decode_kvq8
    one = dict(cu_new=0, max_new=1)
    assert dec(cache(), batch(), P, P, 4, *s, *s, -1.0, 0, 0, 1, None, 0, None) == _lib.ERR_INVALID
    assert dec(cache(), None, P, P, 4, *s, *s, -1.0, 0, 0, 1, None, 0, None) == _lib.ERR_INVALID
    assert dec(None, batch(**one), P, P, 4, *s, *s, -1.0, 0, 0, 1, None, 0, None) == _lib.ERR_INVALID
    assert dec(cache(), batch(**one), P, P, 4, *s, *s, -1.0, 0, 0, 3, None, 0, None) == _lib.ERR_WORKSPACE
    def wb(B, T, new, Hq, H, D, ns, odt=0):
        return L.hipgpt_attn_kvq8_workspace_bytes(B, T, new, Hq, H, D, odt, ns)

    # parts of every row where few rows share a cached head, else two slots of 128 rows a share
    need = wb(2, 2, 1, 4, 2, 64, 3)
    assert need == 2 * 4 * 3 * 66 * 4
    assert dec(cache(), batch(**one), P, P, 4, *s, *s, -1.0, 0, 0, 3, P, need - 4, None) == _lib.ERR_WORKSPACE
    assert dec(cache(), batch(**one), P, P, 4, *s, *s, -1.0, 0, 0, 3, P + 4, need, None) == _lib.ERR_UNSUPPORTED
    assert wb(2, 2, 1, 4, 2, 64, 1) == wb(2, 0, 1, 4, 2, 64, 4) == wb(2, 2, 1, 5, 2, 64, 4) == 0
    assert wb(2, 2, 1, 4, 2, 64, 5000) == wb(2, 2, 1, 4, 2, 64, 1024)
    pre = L.hipgpt_attn_prefill_kvq8
    need = wb(2, 70, 50, 4, 2, 64, 3)
    assert need == 3 * (4 + 2 * 128 * (64 + 4)) * 4
    assert pre(cache(), batch(max_new=50), 70, P, P, 4, *s, *s, -1.0, 0, 0, 3, P, need - 4, None) == _lib.ERR_WORKSPACE
    # 16 rows of a cached head: one tile with a bf16 result, two with an fp32 one, which pay in small batches only
    assert wb(64, 256, 4, 32, 8, 128, 3, 1) == 256 * 32 * 3 * 130 * 4
    assert wb(4, 16, 4, 32, 8, 128, 3, 0) == 16 * 32 * 3 * 130 * 4
    assert wb(64, 256, 4, 32, 8, 128, 3, 0) == 3 * (4 + 2 * 128 * 132) * 4

    def ds(B, T, new, Hq, H, D, ln, odt=0):
        return L.hipgpt_attn_kvq8_default_splits(B, T, new, Hq, H, D, odt, ln)

    assert ds(2, 2, 1, 5, 4, 64, 1 << 20) == 1  # heads that do not divide
    assert ds(0, 2, 1, 4, 4, 64, 99999) == ds(2, 0, 1, 4, 4, 64, 99999) == ds(2, 2, 0, 4, 4, 64, 99999) == 1
    assert ds(1, 1, 1, 8, 8, 64, 1024) == 1
    assert 16 <= ds(1, 1, 1, 8, 8, 64, 1 << 17) <= 256
    assert ds(1, 4096, 4096, 8, 8, 128, 1 << 15) == 512 and ds(64, 65536, 1024, 8, 8, 128, 1024) == 1
    assert ds(1, 500, 500, 8, 8, 128, 1000) == 1


def test_python_wrappers_refuse_host_tensors():
    u8 = torch.zeros(2, 1, 32, 32, dtype=torch.uint8)
    s = torch.ones(2, 1)
    with pytest.raises(TypeError):
        kvcache.CacheQ8(u8, u8, s, s)
    with pytest.raises(TypeError):
        kvcache.Batch(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
