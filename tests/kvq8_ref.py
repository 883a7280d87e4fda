"""64-bit restatement of the paged 8-bit cache (include/hipgpt_attn.h) for its tests: the
byte layout, the rotation, the quantisation of a page and the attention, in numpy."""
import numpy as np

MIN_SCALE = 2.0**-126


def v_bytes(page_size, D):
    """Byte of (token, d) inside a (page, head) of V, [page_size, D], from the header's words:
    [token / 32][D / 32][4][16][2][2][4], token % 32 = 16 i3 + 4 i0 + i4, d % 32 = 16 i2 + i1."""
    at = np.arange(page_size * D).reshape(page_size // 32, D // 32, 4, 16, 2, 2, 4)
    return at.transpose(0, 5, 2, 6, 1, 4, 3).reshape(page_size, D)


def codes_to_pool(codes):
    """Whole numbers c [P, H, ps, D] as the K and V byte pools would hold them."""
    u = (codes + 128).astype(np.uint8)
    P, H, ps, D = u.shape
    v = np.empty_like(u).reshape(P, H, ps * D)
    v[:, :, v_bytes(ps, D).reshape(-1)] = u.reshape(P, H, ps * D)
    return u, v.reshape(P, H, ps, D)


def pool_to_codes(k, v):
    P, H, ps, D = k.shape
    vc = v.reshape(P, H, ps * D)[:, :, v_bytes(ps, D).reshape(-1)].reshape(P, H, ps, D)
    return k.astype(np.int64) - 128, vc.astype(np.int64) - 128


def rotate(x, pos, rot, interleaved, base=10000.0):
    """x [n, H, D] at positions pos, in 64 bits."""
    y = np.array(x, dtype=np.float64)
    if not rot:
        return y
    f = np.float64(base) ** (-2.0 * np.arange(rot // 2) / rot) / (2 * np.pi)
    t = np.asarray(pos, dtype=np.float64)[:, None] * f
    a = 2 * np.pi * (t - np.floor(t))
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    i = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    j = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    x0, x1 = y[..., i].copy(), y[..., j].copy()
    y[..., i], y[..., j] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def attend(q, k, v, G, scale, first):
    """q [n, Hq, D], k, v [N, Hkv, D]: token i sees keys j <= first + i; zeros where none."""
    n, Hq, D = q.shape
    q = q.astype(np.float64)
    out = np.zeros((n, Hq, D))
    for i in range(n):
        m = min(first + i + 1, k.shape[0])
        if m <= 0:
            continue
        for h in range(Hq):
            s = k[:m, h // G] @ q[i, h] * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:m, h // G] / p.sum()
    return out


def f32_tol(v):
    """Error of an fp32 result.  Scores of unit-normal rows stay under ~10 and carry sqrt(D)
    roundings of 2^-24 (D <= 256: 16 * 2^-24 * 10 = 1e-5); a score that is off by e moves the
    result by at most 2 e max|v|."""
    return 2e-5 * np.abs(v).max()


def bf16_tol(o, v):
    """Error of a bf16 result: its rounding (half a step, 2^-8), weights rounded to fp16
    (2^-11), and the fp32 part."""
    return 2.0**-8 * np.abs(o) + 2.0**-11 * np.abs(v).max() + f32_tol(v)
