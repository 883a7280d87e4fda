"""GPU tests of the paged 8-bit cache: append (rotation, page scales, rounding again), read,
decode and prefill, against the 64-bit restatement in kvq8_ref.py.

Pages that no sequence holds have the scale NaN and arbitrary bytes, so reading one would
show; their bytes are compared afterwards, so writing one would too.
"""
import numpy as np
import pytest
import torch

import kvq8_ref as R
from hipgpt_amd import kvcache as K

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def host(t):
    torch.cuda.synchronize()
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def dev_t(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def normal(rng, dtype, *shape):
    """Unit-normal values that `dtype` holds, as the device tensor and in 64 bits."""
    t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DT[dtype])
    return t.cuda(), t.double().numpy()


class Case:
    """A cache of shuffled pages with `cached` tokens per sequence, and spare pages."""

    def __init__(self, seed, cached, room, H, ps, D, pad=0):
        """room: tokens per sequence that the table has pages for.  pad: bytes between pages."""
        rng = self.rng = np.random.default_rng(seed)
        B = len(cached)
        self.cached, self.H, self.ps, self.D = list(cached), H, ps, D
        M = max(1, max(-(-r // ps) for r in room))
        pages = sum(-(-r // ps) for r in room) + 3
        order = rng.permutation(pages)
        self.table = np.full((B, M), -7, dtype=np.int32)
        at = 0
        for b, r in enumerate(room):
            w = -(-r // ps)
            self.table[b, :w] = order[at:at + w]
            at += w
        self.codes = {w: rng.integers(-127, 128, (pages, H, ps, D)) for w in "kv"}
        self.scale = {w: np.full((pages, H), np.nan, dtype=np.float32) for w in "kv"}
        for b, n in enumerate(self.cached):
            for j in range(-(-n // ps)):
                for w in "kv":
                    self.scale[w][self.table[b, j]] = rng.uniform(0.01, 0.03, H)
        ku, vu = R.codes_to_pool(self.codes["k"])[0], R.codes_to_pool(self.codes["v"])[1]
        # pages `pad` bytes apart, scales in a wider array
        buf = torch.from_numpy(rng.integers(0, 256, (2, pages, H * ps * D + pad), dtype=np.uint8)).cuda()
        pools = buf[:, :, :H * ps * D].view(2, pages, H, ps, D)
        pools[0].copy_(torch.from_numpy(ku))
        pools[1].copy_(torch.from_numpy(vu))
        sc = torch.full((2, pages, H + (3 if pad else 0)), float("nan"), device="cuda")
        sc[0, :, :H].copy_(torch.from_numpy(self.scale["k"]))
        sc[1, :, :H].copy_(torch.from_numpy(self.scale["v"]))
        self.cache = K.CacheQ8(pools[0], pools[1], sc[0, :, :H], sc[1, :, :H])
        self.d_table = dev_t(self.table)

    def batch(self, lens, new=None, table=None, max_new=None):
        lens = np.asarray(lens, dtype=np.int32)
        cu = None if new is None else dev_t(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        mn = 1 if new is None else (max_new or max(1, int(max(new))))
        return K.Batch(self.d_table if table is None else table, dev_t(lens), cu, max_new=mn)

    def state(self):
        """Codes and scales as the device holds them now."""
        k, v = R.pool_to_codes(host(self.cache.k), host(self.cache.v))
        return {"k": k, "v": v}, {"k": host(self.cache.k_scale), "v": host(self.cache.v_scale)}

    def rows(self, w, b, n, state=None):
        """The first n tokens of sequence b, [n, H, D] in 64 bits."""
        codes, scale = state or (self.codes, self.scale)
        p = self.table[b, :-(-n // self.ps)]
        x = codes[w][p] * scale[w][p].astype(np.float64)[:, :, None, None]
        return x.transpose(0, 2, 1, 3).reshape(-1, self.H, self.D)[:n]


# ------------------------------------------------------------------------ read


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("ps", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_read_gives_the_values(dev, D, ps, dtype):
    cached = [1, 31, 32, 200, 0, 129]
    c = Case(D + ps, cached, cached, 3, ps, D, pad=48)
    for new in (cached, [1, 0, 5, 131, 0, 129]):
        T = sum(new)
        k, v = K.read(c.cache, c.batch(cached, new), T, dtype=DT[dtype])
        for w, got in (("k", host(k)), ("v", host(v))):
            want = np.concatenate([c.rows(w, b, n)[n - m:] for b, (n, m) in enumerate(zip(cached, new))])
            # one product in fp32 (2^-24), then the output's rounding (bf16 2^-8)
            tol = 2.0**-24 + (2.0**-8 if dtype == "bf16" else 0)
            assert (np.abs(got - want) <= tol * np.abs(want)).all()


# ---------------------------------------------------------------------- append


def check_append(c, lens, new, x, rot, interleaved, before, after):
    """The pages after an append of rows x = {"k", "v"} ([T, H, D], 64 bits, not rotated)."""
    codes0, scale0 = before
    codes1, scale1 = after
    ps = c.ps
    held = np.zeros(c.cache.k.shape[0], dtype=bool)
    at = 0
    for b, (n_all, n) in enumerate(zip(lens, new)):
        first = n_all - n
        pos = np.arange(first, n_all)
        for w in "kv":
            rows = R.rotate(x[w][at:at + n], pos, rot, interleaved) if w == "k" else x[w][at:at + n]
            for j in range(first // ps, -(-n_all // ps) if n else 0):
                page = c.table[b, j]
                held[page] = True
                t0, t1 = max(first - j * ps, 0), min(n_all - j * ps, ps)
                blk = rows[j * ps + t0 - first:j * ps + t1 - first].transpose(1, 0, 2)  # [H, t, D]
                s = scale1[w][page].astype(np.float64)
                want = np.maximum(np.abs(blk).max((1, 2)) / 127, R.MIN_SCALE)
                old = scale0[w][page].astype(np.float64)
                if t0:
                    want = np.maximum(want, old)
                # a rotated value is off by its fp32 products and sum (3 * 2^-24) and its angle
                # (2^-26 turns = 9.4e-8, sine and cosine 2 ulp), of a pair up to sqrt(2) amax: under
                # 1e-6; the division 2^-24
                assert (np.abs(s - want) <= 1.1e-6 * want).all()
                # that error in steps is 127 times it, beside the rounding's half step
                got = codes1[w][page][:, t0:t1]
                assert (np.abs(got - blk / s[:, None, None]) <= 0.5 + 127 * 1.1e-6 + 1e-5).all()
                assert np.abs(got).max() <= 127
                if t0:
                    kept = codes0[w][page][:, :t0]
                    r = (old / s)[:, None, None]
                    got = codes1[w][page][:, :t0]
                    assert np.array_equal(got[s == old], kept[s == old])
                    assert (np.abs(got - kept * r) <= 0.5 + 127 * 2.0**-23).all()
                assert np.array_equal(codes1[w][page][:, t1:], codes0[w][page][:, t1:])  # tokens behind
        at += n
    for w in "kv":
        assert np.array_equal(codes1[w][~held], codes0[w][~held])
        assert np.array_equal(scale1[w][~held], scale0[w][~held], equal_nan=True)


@pytest.mark.parametrize("ps", [32, 64, 128])
@pytest.mark.parametrize("D,rot", [(32, 32), (64, 64), (64, 26), (128, 128), (256, 256), (256, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_ragged(dev, D, rot, ps, interleaved, dtype):
    cached, new = [0, 5, ps - 1, 70, 64, 3], [1, 40, 2, 0, 129, ps]
    lens = [a + b for a, b in zip(cached, new)]
    H, Hq = 2, 6
    c = Case(D + ps + rot, cached, lens, H, ps, D, pad=16)
    T = sum(new)
    q, q64 = normal(c.rng, dtype, T, Hq, D)
    k, k64 = normal(c.rng, dtype, T, H, D)
    v, v64 = normal(c.rng, dtype, T, H, D)
    before = c.state()
    f = K.rope_freqs(rot) if rot else None
    got = host(K.append(c.cache, c.batch(lens, new), q, k, v, freqs=f, interleaved=interleaved))
    check_append(c, lens, new, {"k": k64, "v": v64}, rot, interleaved, before, c.state())
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)])
    want = R.rotate(q64, pos, rot, interleaved)
    # as above for the rotation, of a pair's larger value; bf16 rounds the result (2^-8)
    tol = 1.1e-6 * np.abs(q64).max() + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
    assert (np.abs(got - want) <= tol).all()
    if not rot:
        assert np.array_equal(got, host(q))


def test_append_in_steps_and_far_positions(dev):
    """Token by token into filling pages, steps of growing and shrinking size: the rounding
    again of earlier codes, fresh scales of new pages; positions behind a long prefix."""
    H, ps, D = 2, 32, 64
    room = [300, 100]
    c = Case(11, [250, 0], room, H, ps, D)
    lens = np.array([250, 0])
    f = K.rope_freqs(D)
    for step in range(40):
        lens += 1
        k, k64 = normal(c.rng, "f32", 2, H, D)
        v, v64 = normal(c.rng, "f32", 2, H, D)
        size = 1.0 + 3.0 * (step % 7 == 3)
        before = c.state()
        K.append(c.cache, c.batch(lens), None, k * size, v * size, freqs=f)
        check_append(c, lens, [1, 1], {"k": k64 * size, "v": v64 * size}, D, False, before, c.state())


def test_append_at_a_position_past_a_million(dev):
    """The angle of a far position is exact: 2^20 positions' table, pages shared by one entry."""
    H, ps, D = 1, 128, 128
    n = (1 << 20) + 77
    c = Case(12, [0], [ps], H, ps, D)
    table = torch.full((1, n // ps + 1), int(c.table[0, 0]), dtype=torch.int32, device="cuda")
    q, q64 = normal(c.rng, "f32", 1, 3, D)
    k, _ = normal(c.rng, "f32", 1, H, D)
    got = host(K.append(c.cache, K.Batch(table, dev_t(np.array([n], dtype=np.int32))), q, k, k, freqs=K.rope_freqs(D)))
    want = R.rotate(q64, [n - 1], D, False)
    # the reference's own angle: position times a 2^-53 rounding of the frequency
    assert np.abs(got - want).max() <= 1.1e-6 * np.abs(q64).max() + 2 * np.pi * n * 0.16 * 2.0**-52 * 4


def test_append_in_place_strided_and_on_a_stream(dev):
    """q, k, v as column windows of one projection output, q rotated in place, on another stream."""
    H, ps, D = 4, 64, 64
    lens, new = [70, 3], [66, 3]
    c = Case(13, [4, 0], lens, H, ps, D)
    qkv, x64 = normal(c.rng, "bf16", sum(new), 3, H, D)
    q, k, v = (qkv[:, i] for i in range(3))
    before = c.state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = K.append(c.cache, c.batch(lens, new), q, k, v, freqs=K.rope_freqs(D), q_out=q, stream=s)
    s.synchronize()
    assert out.data_ptr() == q.data_ptr()
    check_append(c, lens, new, {"k": x64[:, 1], "v": x64[:, 2]}, D, False, before, c.state())
    pos = np.concatenate([np.arange(4, 70), np.arange(3)])
    want = R.rotate(x64[:, 0], pos, D, False)
    assert (np.abs(host(q) - want) <= 1.1e-6 * 5 + 2.0**-8 * np.abs(want)).all()
    assert np.array_equal(host(qkv[:, 1:]), x64[:, 1:])  # k and v only read


def test_append_odd_values(dev):
    """Zeros, the smallest and largest numbers, infinities and NaN: scales as documented."""
    H, ps, D = 6, 32, 32
    c = Case(14, [0], [3], H, ps, D)
    x = np.zeros((3, H, D), dtype=np.float32)
    x[1, 1, 4] = 1e-45
    x[:, 2] = 3e38
    x[2, 2] = -3.4e38
    x[1, 3, 5] = np.inf
    x[0, 4, 0] = np.nan
    x[:, 5, 7] = 2.0
    K.append(c.cache, c.batch([3], [3]), None, dev_t(x), dev_t(x))
    codes, scale = c.state()
    page = c.table[0, 0]
    for w in "kv":
        s = scale[w][page]
        assert s[0] == s[1] == np.float32(R.MIN_SCALE)
        assert np.isnan(s[3]) and np.isnan(s[4]) and s[5] == np.float32(2.0) / np.float32(127)
        assert not codes[w][page, :2, :3].any()
        assert (codes[w][page, 2, :2] == round(3e38 / 3.4e38 * 127)).all() and (codes[w][page, 2, 2] == -127).all()
        assert (codes[w][page, 5, :3, 7] == 127).all()
    # a page stays NaN while it fills, and a new page starts afresh
    c2 = Case(15, [0], [64], 1, ps, D)
    x = np.ones((40, 1, D), dtype=np.float32)
    x[3] = np.nan
    K.append(c2.cache, c2.batch([20], [20]), None, dev_t(x[:20]), dev_t(x[:20]))
    K.append(c2.cache, c2.batch([40], [20]), None, dev_t(x[20:]), dev_t(x[20:]))
    _, scale = c2.state()
    assert np.isnan(scale["k"][c2.table[0, 0]]) and scale["v"][c2.table[0, 1]] == np.float32(1) / np.float32(127)


def test_append_refuses_on_the_device(dev):
    """Bad lengths, page indexes and row ranges: nothing is stored, the others go on."""
    H, ps, D = 2, 32, 32
    lens, new = [-1, 3, 500, 40, 2, 7], [2, 5, 2, 2, 2, 7]
    c = Case(16, [0] * 6, [40] * 6, H, ps, D)
    c.table[3, 1] = 10**6  # holds token 38, 39
    c.table[4, 0] = -1
    c.d_table = dev_t(c.table)
    T = sum(new)
    q, _ = normal(c.rng, "f32", T, H, D)
    k, k64 = normal(c.rng, "f32", T, H, D)
    v, v64 = normal(c.rng, "f32", T, H, D)
    before = c.state()
    got = host(K.append(c.cache, c.batch(lens, new), q, k, v, freqs=K.rope_freqs(D)))
    after = c.state()
    c.table[:5] = 0  # only the last sequence is held to the check
    check_append(c, [0] * 5 + [7], [0] * 5 + [7], {"k": k64[-7:], "v": v64[-7:]}, D, False, before, after)
    assert np.isnan(got[:2]).all() and np.isnan(got[2:9]).all() and np.isfinite(got[9:]).all()
    # row ranges outside the packed rows, or running backwards: no row of theirs is touched
    cu = dev_t(np.array([0, 2, 1, 4, 9, 9, T + 1], dtype=np.int32))
    out = torch.full((T, H, D), 77.0, device="cuda")
    before = c.state()
    K.append(c.cache, K.Batch(c.d_table, dev_t(np.array([2, 9, 3, 5, 0, 7], dtype=np.int32)), cu, max_new=5), q, k, v,
             q_out=out)
    after = c.state()
    got = host(out)
    assert (got[9:] == 77.0).all() and (got[:9] != 77.0).any()
    assert np.array_equal(after[0]["k"][c.table[5, 0]], before[0]["k"][c.table[5, 0]])


def test_advance(dev):
    c = Case(17, [5, 0, 30], [64] * 3, 1, 32, 32)
    k, _ = normal(c.rng, "f32", 3, 1, 32)
    b = c.batch([5, 0, 30])
    K.append(c.cache, b, None, k, k, advance=True)
    assert host(b.lens).tolist() == [6, 1, 31]
    b2 = K.Batch(c.d_table, b.lens, dev_t(np.array([0, 0, 1, 3], dtype=np.int32)), max_new=2)
    K.append(c.cache, b2, None, k, k, advance=True)
    assert host(b.lens).tolist() == [6, 2, 33]
    # a slot without a sequence stays one, and nothing is stored for it
    b3 = c.batch([6, -1, 2**31 - 1])
    before = c.state()
    K.append(c.cache, b3, None, k, k, advance=True)
    assert host(b3.lens).tolist() == [7, -1, 2**31 - 1]
    for w in "kv":
        assert np.array_equal(c.state()[0][w][c.table[1:]], before[0][w][c.table[1:]])


# ------------------------------------------------------------------- attention


def check_attention(c, got, q64, lens, new, G, scale, out, state=None, skip=()):
    at = 0
    for b, (n_all, n) in enumerate(zip(lens, new)):
        if b in skip:
            at += n
            continue
        k, v = c.rows("k", b, n_all, state), c.rows("v", b, n_all, state)
        want = R.attend(q64[at:at + n], k, v, G, scale, n_all - n)
        if n and n_all:
            tol = R.f32_tol(v) if out == "f32" else R.bf16_tol(want, v)
            assert (np.abs(got[at:at + n] - want) <= tol).all(), (b, np.abs(got[at:at + n] - want).max())
        else:
            assert (got[at:at + n] == 0).all()
        at += n


TYPES = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")]


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("ps", [32, 64, 128])
@pytest.mark.parametrize("G", [1, 3, 8, 20])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_decode(dev, D, ps, G, dtype, out):
    lens = [1, 31, 0, 32, 33, 257, 130, 64]
    H = 2
    c = Case(D * ps + G, lens, lens, H, ps, D, pad=32)
    q, q64 = normal(c.rng, dtype, len(lens), G * H, D)
    for splits in (1, None, 3):
        got = host(K.decode(c.cache, c.batch(lens), q, out_dtype=DT[out], num_splits=splits))
        check_attention(c, got, q64, lens, [1] * len(lens), G, D**-0.5, out)


@pytest.mark.parametrize("splits", [1, None, 64])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_decode_long(dev, splits, dtype, out):
    """A few thousand keys, and more splits than some sequences have tiles."""
    lens = [5000, 40]
    c = Case(21, lens, lens, 2, 64, 128)
    q, q64 = normal(c.rng, dtype, 2, 8, 128)
    got = host(K.decode(c.cache, c.batch(lens), q, out_dtype=DT[out], num_splits=splits, scale=0.3))
    check_attention(c, got, q64, lens, [1, 1], 4, 0.3, out)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("G", [1, 4, 7])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_prefill(dev, D, G, dtype, out):
    cached, new = [0, 100, 1, 63, 7, 300], [70, 33, 0, 1, 129, 17]
    lens = [a + b for a, b in zip(cached, new)]
    H, ps = 2, 64
    c = Case(D + G, lens, lens, H, ps, D, pad=16)
    q, q64 = normal(c.rng, dtype, sum(new), G * H, D)
    for splits in (1, 3, 40, None):
        got = host(K.prefill(c.cache, c.batch(lens, new), q, out_dtype=DT[out], num_splits=splits))
        check_attention(c, got, q64, lens, new, G, D**-0.5, out)


@pytest.mark.parametrize("ps", [32, 128])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_prefill_long_chunk(dev, ps, dtype, out):
    """Rows of several blocks behind a prefix that is no multiple of a tile; strided q and out."""
    cached, new = [513, 0], [300, 257]
    lens = [a + b for a, b in zip(cached, new)]
    H, D = 1, 64
    c = Case(31, lens, lens, H, ps, D)
    T = sum(new)
    wide, w64 = normal(c.rng, dtype, T, 3, 2, D)
    buf = torch.full((T, 4, D + 8), 5.0, device="cuda", dtype=DT[out])
    got = K.prefill(c.cache, c.batch(lens, new, max_new=400), wide[:, 1], out=buf[:, 1:3, :D])
    check_attention(c, host(got), w64[:, 1], lens, new, 2, D**-0.5, out)
    assert (buf[:, [0, 3]] == 5).all() and (buf[:, :, D:] == 5).all()


def test_prefill_equals_decode_for_single_tokens(dev):
    lens = [5, 130, 64]
    c = Case(41, lens, lens, 2, 32, 64)
    q, q64 = normal(c.rng, "f32", 3, 4, 64)
    a = host(K.decode(c.cache, c.batch(lens), q))
    b = host(K.prefill(c.cache, c.batch(lens, [1, 1, 1]), q))
    for got in (a, b):
        check_attention(c, got, q64, lens, [1] * 3, 2, 0.125, "f32")


@pytest.mark.parametrize("call", ["decode", "prefill"])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_peaked_scores_and_uneven_scales(dev, call, dtype, out):
    """One key holds all the weight; page scales a thousandfold apart; q of large size."""
    n, H, ps, D = 200, 1, 32, 64
    c = Case(51, [n], [n], H, ps, D)
    for j, p in enumerate(c.table[0, :-(-n // ps)]):
        c.scale["v"][p] = 1e-3 if j % 2 else 1.0
        c.scale["k"][p] = 0.02
    c.cache.k_scale.copy_(torch.from_numpy(c.scale["k"]))
    c.cache.v_scale.copy_(torch.from_numpy(c.scale["v"]))
    q, q64 = normal(c.rng, dtype, 1, 2, D)
    for size in (1.0, 30.0, 1e-20):
        qs = (q * size).to(q.dtype)
        q64 = qs.double().cpu().numpy()
        b = c.batch([n]) if call == "decode" else c.batch([n], [1])
        got = host(getattr(K, call)(c.cache, b, qs, out_dtype=DT[out]))
        k, v = c.rows("k", 0, n), c.rows("v", 0, n)
        want = R.attend(q64, k, v, 2, D**-0.5, n - 1)
        # at size 30 scores reach ~300: sqrt(64) roundings of 2^-24 of them, twice in the result
        far = 2 * 8 * 2.0**-24 * 300 * np.abs(v).max()
        tol = (R.f32_tol(v) if out == "f32" else R.bf16_tol(want, v)) + far
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_attention_bad_sequences(dev, call):
    """Bad lengths and pages give NaN rows, the others are right; a NaN page that a row does
    not see leaves it alone; NaN and infinite queries stay in their rows."""
    H, ps, D, G = 2, 32, 64, 2
    lens = [40, -3, 1000, 50, 33, 20]
    c = Case(61, [40, 0, 0, 50, 33, 20], [96] * 6, H, ps, D)
    c.table[3, 1] = 9999
    c.d_table = dev_t(c.table)
    q, q64 = normal(c.rng, "f32", 6, G * H, D)
    q[5, 1, 3] = float("nan")
    q[5, 2, 0] = float("inf")
    new = [1] * 6
    b = c.batch(lens) if call == "decode" else c.batch(lens, new)
    for kw in ({}, {"num_splits": 3}):
        got = host(getattr(K, call)(c.cache, b, q, **kw))
        check_attention(c, got, q64, lens, new, G, 0.125, "f32", skip=(1, 2, 3, 5))
        assert np.isnan(got[1:4]).all() and np.isnan(got[5, 1:3]).all()
        k, v = c.rows("k", 5, 20), c.rows("v", 5, 20)
        want = R.attend(q64[5:], k, v, G, 0.125, 19)
        assert np.abs(got[5, [0, 3]] - want[0, [0, 3]]).max() <= R.f32_tol(v)


@pytest.mark.parametrize("dtype,out", TYPES)
def test_prefill_does_not_see_what_is_behind(dev, dtype, out):
    """A page with the scale NaN poisons the rows that see it, and no earlier one."""
    H, ps, D = 1, 32, 32
    n = 96
    c = Case(71, [n], [n], H, ps, D)
    c.cache.v_scale[int(c.table[0, 2])] = float("nan")
    c.cache.k_scale[int(c.table[0, 1])] = float("nan")
    q, q64 = normal(c.rng, dtype, n, 2, D)
    k, v = c.rows("k", 0, 32), c.rows("v", 0, 32)
    want = R.attend(q64[:32], k, v, 2, D**-0.5, 0)
    tol = R.f32_tol(v) if out == "f32" else R.bf16_tol(want, v)
    for splits in (1, 3):
        got = host(K.prefill(c.cache, c.batch([n], [n]), q, out_dtype=DT[out], num_splits=splits))
        assert np.isnan(got[32:]).all()
        assert (np.abs(got[:32] - want) <= tol).all()


def test_rows_that_no_sequence_names_stay(dev):
    lens, new = [40, 9], [5, 3]
    c = Case(81, lens, lens, 1, 32, 64)
    q, q64 = normal(c.rng, "bf16", 12, 2, 64)
    out = torch.full((12, 2, 64), 3.0, device="cuda")
    K.prefill(c.cache, c.batch(lens, new), q, out=out)
    check_attention(c, host(out)[:8], q64, lens, new, 2, 0.125, "f32")
    assert (out[8:] == 3).all()
    k = torch.full((12, 1, 64), 4.0, device="cuda")
    K.read(c.cache, c.batch(lens, new), 12, k=k, v=k.clone())
    assert (k[8:] == 4).all() and (k[:8] != 4).any()


def test_offsets_past_32_bits(dev):
    """A pool of more than 4 GiB: the last pages are addressed in 64 bits."""
    H, ps, D = 8, 128, 256
    pages = (4 << 30) // (H * ps * D) + 40
    codes = torch.zeros(2, pages, H, ps, D, dtype=torch.uint8, device="cuda")
    cache = K.CacheQ8(codes[0], codes[1], *torch.full((2, pages, H), float("nan"), device="cuda"))
    n = 200
    table = dev_t(np.array([[pages - 1, pages - 30]], dtype=np.int32))
    rng = np.random.default_rng(5)
    k, k64 = normal(rng, "f32", n, H, D)
    v, v64 = normal(rng, "f32", n, H, D)
    q, q64 = normal(rng, "f32", n, H, D)
    b = K.Batch(table, dev_t(np.array([n], dtype=np.int32)), dev_t(np.array([0, n], dtype=np.int32)), max_new=n)
    K.append(cache, b, None, k, v)
    rk, rv = (host(x).astype(np.float64) for x in K.read(cache, b, n))
    # a code is off by half a step of max / 127
    assert np.abs(rk - k64).max() <= np.abs(k64).max() / 253 and np.abs(rv - v64).max() <= np.abs(v64).max() / 253
    one = K.Batch(table, b.lens)
    got = host(K.decode(cache, one, q[-1:].contiguous(), num_splits=2))
    want = R.attend(q64[-1:], rk, rv, 1, 1 / 16, n - 1)
    assert np.abs(got - want).max() <= R.f32_tol(rv)
    got = host(K.prefill(cache, b, q))[-3:]
    want = R.attend(q64[-3:], rk, rv, 1, 1 / 16, n - 3)
    assert np.abs(got - want).max() <= R.f32_tol(rv)


# ------------------------------------------------------------------- together


@pytest.mark.parametrize("dtype,out", TYPES)
def test_serving_run(dev, dtype, out):
    """Prompts in two ragged chunks, then generated tokens, with append / prefill / decode as a
    program calls them (lengths advanced on the device): each step's rows against the 64-bit
    attention over the values that the cache holds, and those against the tokens given."""
    H, G, ps, D = 2, 3, 32, 64
    c = Case(91, [0, 0, 0], [200, 90, 40], H, ps, D)
    f = K.rope_freqs(D)
    lens = np.zeros(3, dtype=np.int64)
    d_lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    given = {w: [np.zeros((0, H, D)) for _ in range(3)] for w in "kv"}
    for new in [[100, 33, 0], [61, 0, 17]] + [None] * 5:
        n = [1, 1, 1] if new is None else new
        T = sum(n)
        q, q64 = normal(c.rng, dtype, T, G * H, D)
        k, k64 = normal(c.rng, dtype, T, H, D)
        v, v64 = normal(c.rng, dtype, T, H, D)
        cu = None if new is None else dev_t(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        b = K.Batch(c.d_table, d_lens, cu, max_new=max(n))
        qr = K.append(c.cache, b, q, k, v, freqs=f, advance=True)
        lens += n
        got = host((K.decode if new is None else K.prefill)(c.cache, b, qr, out_dtype=DT[out]))
        assert np.array_equal(host(d_lens), lens)
        qr = host(qr).astype(np.float64)
        state = c.state()
        check_attention(c, got, qr, lens, n, G, D**-0.5, out, state)
        at = 0
        for s in range(3):
            pos = np.arange(lens[s] - n[s], lens[s])
            given["k"][s] = np.concatenate([given["k"][s], R.rotate(k64[at:at + n[s]], pos, D, False)])
            given["v"][s] = np.concatenate([given["v"][s], v64[at:at + n[s]]])
            at += n[s]
            for w in "kv":
                x = given[w][s]
                if len(x):
                    # half a step of the page's scale, again for each time that it grew: at most 8 here
                    p = c.table[s, np.arange(len(x)) // ps]
                    step = state[1][w][p][:, :, None].astype(np.float64)
                    assert (np.abs(c.rows(w, s, len(x), state) - x) <= 4 * step).all()


def test_captured_steps_replay(dev):
    """A decode step (append with advance, decode in splits, then a prefill of the same row)
    captured once and replayed: every replay equals the eager step on a copy of its state, with
    eager work of the program in between."""
    H, ps, D, B = 2, 32, 64, 3
    c = Case(95, [40, 7, 0], [200] * 3, H, ps, D)
    f = K.rope_freqs(D)
    q, k, v = (normal(c.rng, "f32", B, H, D)[0] for _ in range(3))
    out, out2, qr = (torch.empty(B, H, D, device="cuda") for _ in range(3))
    ws = torch.empty(K.workspace_bytes(B, B, 1, H, H, D, torch.float32, 4), dtype=torch.uint8, device="cuda")
    lens = dev_t(np.array([40, 7, 0], dtype=np.int32))
    cu = dev_t(np.arange(B + 1, dtype=np.int32))

    def step(cache, lens):
        b = K.Batch(c.d_table, lens)
        K.append(cache, b, q, k, v, freqs=f, q_out=qr, advance=True)
        K.decode(cache, b, qr, out=out, num_splits=4, workspace=ws)
        K.prefill(cache, K.Batch(c.d_table, lens, cu), qr, out=out2)

    def copy():
        t = c.cache
        return K.CacheQ8(t.k.clone(), t.v.clone(), t.k_scale.clone(), t.v_scale.clone()), lens.clone()

    step(*copy())  # eager once before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(c.cache, lens)
    torch.cuda.synchronize()
    for i in range(6):
        for x in (q, k, v):
            x.copy_(normal(c.rng, "f32", B, H, D)[0])
        cache2, lens2 = copy()
        step(cache2, lens2)  # eager, on a copy
        want = [t.clone() for t in (out, out2, qr, cache2.k, cache2.v, cache2.k_scale, cache2.v_scale, lens2)]
        for t in (out, out2, qr):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = (out, out2, qr, c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale, lens)
        for a, b in zip(got, want):
            assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a,
                               b.nan_to_num(7.0) if b.is_floating_point() else b), i


def test_same_inputs_give_the_same_bits(dev):
    lens, new = [700, 90], [300, 11]
    c = Case(97, lens, lens, 2, 64, 128)
    q, _ = normal(c.rng, "f32", sum(new), 4, 128)
    a = K.prefill(c.cache, c.batch(lens, new), q)
    b = K.decode(c.cache, c.batch(lens), q[:2].contiguous(), num_splits=5)
    for _ in range(3):
        assert torch.equal(K.prefill(c.cache, c.batch(lens, new), q), a)
        assert torch.equal(K.decode(c.cache, c.batch(lens), q[:2].contiguous(), num_splits=5), b)


def test_wrappers_refuse(dev):
    c = Case(99, [5], [5], 2, 32, 64)
    b = c.batch([5])
    q = torch.zeros(1, 4, 64, device="cuda")
    with pytest.raises(ValueError):
        K.decode(c.cache, b, torch.zeros(2, 4, 64, device="cuda"))  # rows of another batch
    with pytest.raises(ValueError):
        K.decode(c.cache, b, torch.zeros(1, 4, 32, device="cuda"))
    with pytest.raises(TypeError):
        K.decode(c.cache, b, q.half())
    with pytest.raises(Exception):
        K.decode(c.cache, b, q, out_dtype=torch.bfloat16)  # fp32 q, bf16 out
    with pytest.raises(Exception):
        K.decode(c.cache, b, torch.zeros(1, 3, 64, device="cuda"))  # heads that do not divide
    with pytest.raises(TypeError):
        K.append(c.cache, b, None, q[:, :2].bfloat16(), q[:, :2])
    with pytest.raises(ValueError):
        K.Batch(c.d_table, b.lens, None, max_new=3)
    with pytest.raises(ValueError):
        K.append(c.cache, b, None, q[:, :2], q[:, :2], q_out=q)


def test_empty_slots(dev):
    """lens[b] = 0 in a batch of single tokens: nothing stored, nothing read, zeros."""
    c = Case(101, [0, 4, 0], [32] * 3, 2, 32, 64)
    q, q64 = normal(c.rng, "f32", 3, 4, 64)
    k, k64 = normal(c.rng, "f32", 3, 2, 64)
    before = c.state()
    b = c.batch([0, 5, 0])
    K.append(c.cache, b, q, k, k)
    after = c.state()
    for s in (0, 2):
        for w in "kv":
            assert np.array_equal(after[0][w][c.table[s, 0]], before[0][w][c.table[s, 0]])
    rows = torch.full((3, 2, 64), 9.0, device="cuda")
    K.read(c.cache, b, 3, k=rows, v=rows.clone())
    assert (rows[[0, 2]] == 9).all() and (rows[1] != 9).any()
    for splits in (1, 2):
        got = host(K.decode(c.cache, b, q, num_splits=splits))
        assert not got[[0, 2]].any()
        kk, vv = (after[0][w][c.table[1, 0]] * after[1][w][c.table[1, 0]].astype(np.float64)[:, None, None]
                  for w in "kv")
        want = R.attend(q64[1:2], kk.transpose(1, 0, 2)[:5], vv.transpose(1, 0, 2)[:5], 2, 0.125, 4)
        assert np.abs(got[1:2] - want).max() <= R.f32_tol(vv)


@pytest.mark.parametrize("splits", [1, 7])
def test_captured_prefill_replays(dev, splits):
    """The 128-row blocks (whole and in shares) captured with an append: replays equal the eager
    calls, with eager work of the program in between."""
    H, ps, D, n = 2, 64, 128, 150
    c = Case(111, [300, 20], [600, 200], H, ps, D)
    lens, new = [300 + n, 20 + 60], [n, 60]
    b = c.batch(lens, new)
    q, k, v = (normal(c.rng, "bf16", sum(new), h, D)[0] for h in (4, H, H))
    qr, out = torch.empty_like(q), torch.empty(sum(new), 4, D, device="cuda")
    need = K.workspace_bytes(2, sum(new), n, 4, H, D, torch.float32, splits)
    ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    f = K.rope_freqs(D)

    def step():
        K.append(c.cache, b, q, k, v, freqs=f, q_out=qr)
        K.prefill(c.cache, b, qr, out=out, num_splits=splits, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    torch.cuda.synchronize()
    for i in range(4):
        step()  # appending the same rows again leaves the codes as they are
        want = out.clone()
        out.fill_(float("nan"))
        ws.fill_(255)  # what a workspace holds before a call does not matter
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    check_attention(c, host(out), host(qr).astype(np.float64), lens, new, 2, D**-0.5, "f32", c.state())


def test_streams_at_once(dev):
    """Decode and prefill of two batches over one cache on two streams, workspaces of their own."""
    lens = [1500, 900]
    c = Case(121, lens, lens, 2, 64, 64)
    q1, q64 = normal(c.rng, "f32", 2, 8, 64)
    q2, p64 = normal(c.rng, "f32", 130, 8, 64)
    new = [100, 30]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    b1, b2 = c.batch(lens), c.batch(lens, new)
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got.append((K.decode(c.cache, b1, q1, num_splits=6, stream=s1),
                    K.prefill(c.cache, b2, q2, num_splits=9, stream=s2)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, got[0][0]) and torch.equal(b, got[0][1])
    check_attention(c, host(got[0][0]), q64, lens, [1, 1], 4, 0.125, "f32")
    check_attention(c, host(got[0][1]), p64, lens, new, 4, 0.125, "f32")


@pytest.mark.parametrize("dtype,out", TYPES)
def test_mixed_batch_and_wide_tables(dev, dtype, out):
    """Prompts beside single tokens and idle sequences; a table wider than its rows use."""
    cached, new = [0, 500, 40, 7, 0], [200, 1, 0, 1, 33]
    lens = [a + b for a, b in zip(cached, new)]
    c = Case(131, lens, lens, 2, 32, 64)
    wide = torch.full((5, c.table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.d_table
    q, q64 = normal(c.rng, dtype, sum(new), 4, 64)
    for splits in (1, 5):
        b = c.batch(lens, new, table=wide[:, :c.table.shape[1]])
        got = host(K.prefill(c.cache, b, q, out_dtype=DT[out], num_splits=splits))
        check_attention(c, got, q64, lens, new, 2, 0.125, out)


@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_zero_and_tiny_values(dev, call):
    """Pages of zeros (scale 2^-126) among others: they count in the sums and add nothing."""
    n, H, ps, D = 130, 1, 32, 64
    c = Case(141, [n], [n], H, ps, D)
    for j in (0, 2):
        for w in "kv":
            c.scale[w][c.table[0, j]] = np.float32(R.MIN_SCALE)
    c.cache.k_scale.copy_(torch.from_numpy(c.scale["k"]))
    c.cache.v_scale.copy_(torch.from_numpy(c.scale["v"]))
    q, q64 = normal(c.rng, "f32", 1, 2, D)
    wide = q.expand(1, 2, D).repeat(1, 20, 1)  # 40 rows of one head: the 128-row blocks in prefill
    b = c.batch([n]) if call == "decode" else c.batch([n], [1])
    got = host(getattr(K, call)(c.cache, b, wide))
    k, v = c.rows("k", 0, n), c.rows("v", 0, n)
    want = np.tile(R.attend(q64, k, v, 2, 0.125, n - 1), (1, 20, 1))
    assert np.abs(got - want).max() <= R.f32_tol(v)


def test_pools_by_head(dev):
    """Pools laid out [heads][pages] and scales likewise, seen as [pages, heads]."""
    lens, new = [70, 33], [70, 3]
    c = Case(151, [0, 30], lens, 3, 32, 64)
    t = c.cache
    codes = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (t.k, t.v)]
    scales = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (t.k_scale, t.v_scale)]
    c.cache = K.CacheQ8(*codes, *scales)
    q, q64 = normal(c.rng, "bf16", 73, 6, 64)
    k, k64 = normal(c.rng, "bf16", 73, 3, 64)
    v, v64 = normal(c.rng, "bf16", 73, 3, 64)
    before = c.state()
    K.append(c.cache, c.batch(lens, new), None, k, v)
    check_append(c, lens, new, {"k": k64, "v": v64}, 0, False, before, c.state())
    got = host(K.prefill(c.cache, c.batch(lens, new), q))
    check_attention(c, got, q64, lens, new, 2, 0.125, "f32", c.state())


def test_workspace_refusals(dev):
    c = Case(161, [2000], [2000], 2, 64, 64)
    q, _ = normal(c.rng, "f32", 1, 2, 64)
    need = K.workspace_bytes(1, 1, 1, 2, 2, 64, torch.float32, 4)
    ws = torch.empty(2 * need, dtype=torch.uint8, device="cuda")
    b = c.batch([2000])
    for bad in (torch.empty(need, dtype=torch.uint8), ws[::2]):
        with pytest.raises(ValueError, match="workspace"):
            K.decode(c.cache, b, q, num_splits=4, workspace=bad)
    with pytest.raises(Exception, match="(?i)workspace"):
        K.decode(c.cache, b, q, num_splits=4, workspace=ws[:need - 1])


def test_table_past_int_tokens(dev):
    """A table whose row holds 2^31 tokens and more, and a max_len beyond int: the default split."""
    c = Case(162, [2900], [2900], 2, 128, 64)
    q, q64 = normal(c.rng, "f32", 1, 2, 64)
    table = torch.zeros(1, (1 << 24) + 1, dtype=torch.int32, device="cuda")
    table[0, :c.table.shape[1]] = torch.from_numpy(c.table[0]).cuda()
    lens = torch.tensor([2900], dtype=torch.int32, device="cuda")
    k, v = c.rows("k", 0, 2900), c.rows("v", 0, 2900)
    want = R.attend(q64, k, v, 1, 0.125, 2899)
    for max_len in (None, 1 << 31, 1 << 33):
        got = host(K.decode(c.cache, K.Batch(table, lens, max_len=max_len), q))
        assert np.abs(got - want).max() <= R.f32_tol(v)
