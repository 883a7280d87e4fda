"""The paged 8-bit key/value cache and the attention over it, as cases to measure.

``run`` computes each operator in its plain form (elementary torch operations in
32 bits), or with ``own`` set through ``hipgpt_amd.kvcache``.  A case's ``kind``:

* ``append``  -- rotate the new tokens' q and k by their position, quantise k and v
  into the pages, and read the pages that were touched back as values.
* ``read``    -- the values that all cached tokens of a batch stand for.
* ``decode``  -- one query row per sequence against its cached tokens.
* ``prefill`` -- a ragged chunk of new tokens per sequence, causal against the cache
  (which already holds the chunk).

The cache: pages of ``page`` tokens; per (page, head) one scale for K and one for V;
a value is (code - 128) * scale, codes 1..255.  K codes are [page, head, token, D];
V codes [page, head, token / 32, D / 32, 4, 16, 2, 2, 4], where token % 32 is
16 i3 + 4 i0 + i4 and d % 32 is 16 i2 + i1 of the last five indexes i0..i4.
"""
import math
import random

import torch

own = False


# ------------------------------------------------------------------- cases


def _case(name, kind, B, Hq, Hkv, D, page, dtype, out, new, cached, rot=None, interleaved=False, base=10000.0):
    """``new``: (fewest, most) new tokens of a sequence; ``cached``: (fewest, most)
    tokens that it holds before them.  ``dtype``: of q, k, v; ``out``: of the result."""
    return {"name": name, "kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "out": out,
            "new_lo": new[0], "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1],
            "rot": D if rot is None else rot, "interleaved": interleaved, "base": base}


def listed():
    return [
        # one generated token of one sequence, a GPT-2-small layer's heads: the smallest append
        _case("append_one", "append", 1, 12, 12, 64, 64, "f32", "bf16", (1, 1), (700, 700)),
        # a serving step's append: 64 sequences of all lengths, four query heads to a cached head
        _case("append_step", "append", 64, 32, 8, 128, 64, "bf16", "bf16", (1, 1), (0, 8191), base=500000.0),
        # prompts of odd lengths going into the cache, some behind what is there already
        _case("append_prompts", "append", 8, 16, 16, 128, 64, "bf16", "bf16", (901, 2048), (0, 77), interleaved=True),
        # short sequences read back, the default model's heads
        _case("read_short", "read", 5, 8, 8, 32, 32, "f32", "f32", (0, 0), (1, 999)),
        # long sequences handed over to a bf16 consumer
        _case("read_long", "read", 8, 8, 8, 128, 128, "bf16", "bf16", (0, 0), (6001, 8192)),
        # one token of one short sequence: latency
        _case("decode_one", "decode", 1, 12, 12, 64, 64, "f32", "f32", (1, 1), (332, 332)),
        # a generation step of a GPT-2-small layer, sequences of all lengths up to 2048
        _case("decode_gpt2", "decode", 64, 12, 12, 64, 64, "f32", "f32", (1, 1), (0, 2047)),
        # a serving step over long contexts, grouped heads, bf16 in and out
        _case("decode_grouped", "decode", 64, 32, 8, 128, 64, "bf16", "bf16", (1, 1), (511, 8191)),
        # two very long sequences: few rows, the keys have to be split
        _case("decode_long", "decode", 2, 32, 8, 128, 128, "bf16", "f32", (1, 1), (65536, 131071)),
        # prompts of a GPT-2-small layer from an empty cache, fp32
        _case("prefill_gpt2", "prefill", 8, 12, 12, 64, 64, "f32", "f32", (1024, 1024), (0, 0)),
        # chunks of odd lengths behind long cached prefixes, grouped heads
        _case("prefill_chunk", "prefill", 4, 32, 8, 128, 64, "bf16", "bf16", (133, 512), (3999, 8000)),
        # whole prompts at the larger head dim
        _case("prefill_long", "prefill", 4, 16, 16, 128, 64, "bf16", "bf16", (2048, 2048), (0, 0)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# The most that a drawn case may ask for: (bytes, flops) of one pass.
_LIMIT = {"append": (9.0e7, 1e18), "read": (1.5e8, 1e18), "decode": (4.0e8, 1e18), "prefill": (3.0e8, 5.0e10)}


def draw(rng):
    while True:
        kind = rng.choice(sorted(_LIMIT))
        D = rng.choice([32, 64, 64, 128, 128, 256])
        Hkv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        G = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        B = _log_int(rng, 1, 96)
        new = (1, 1)
        if kind == "read":
            new = (0, 0)
        elif kind == "prefill" or (kind == "append" and rng.random() < 0.5):
            hi = _log_int(rng, 2, 2048)
            new = (rng.randint(0 if B > 1 else 1, hi), hi)
        hi = _log_int(rng, 1, 32768)
        cached = (rng.randint(0, hi), hi) if rng.random() < 0.8 else (0, 0)
        if kind == "read" and cached[1] == 0:
            cached = (1, hi)
        rot = D if rng.random() < 0.7 else rng.randint(1, D // 2) * 2
        dtype, out = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
        if kind == "append":
            out = "bf16"
        case = _case("", kind, B, G * Hkv, Hkv, D, rng.choice([32, 64, 128]), dtype, out, new, cached, rot,
                     rng.random() < 0.5, rng.choice([10000.0, 500000.0]))
        del case["name"]
        w = work(case)
        lens, n_new = _lens(case)
        # what the plain form of the attention holds: K and V in 32 bits, and its scores
        dense, scores = B * max(lens) * Hkv * D, B * G * Hkv * max(n_new) * max(lens)
        if w["bytes"] > _LIMIT[kind][0] or w["flops"] > _LIMIT[kind][1] or (kind != "read" and not sum(n_new)):
            continue
        if kind not in ("decode", "prefill") or (dense <= 1.2e9 and scores <= 6e8):
            return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi in a mixed order, both ends among them."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _lens(case):
    """Tokens of each sequence with the new ones, and the new ones alone."""
    new = _spread(case["new_lo"], case["new_hi"], case["B"])
    cached = _spread(case["cached_lo"], case["cached_hi"], case["B"])[::-1]
    return [c + n for c, n in zip(cached, new)], new


def _touched(case):
    """Tokens of each sequence from the start of the first page that an append writes to."""
    lens, new = _lens(case)
    return [n_all - (n_all - n) // case["page"] * case["page"] if n else 0 for n_all, n in zip(lens, new)]


def work(case):
    lens, new = _lens(case)
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    el, out = (4 if case["dtype"] == "f32" else 2), (4 if case["out"] == "f32" else 2)
    T = sum(new)
    pages = lambda ns: sum(-(-n // ps) for n in ns)  # noqa: E731
    if case["kind"] == "append":
        back = _touched(case)
        # q in and out, k and v in, their codes and scales out; then the pages back
        nbytes = T * D * (2 * Hq * el + 2 * Hkv * (el + 1)) + 8 * Hkv * pages(back)
        nbytes += 2 * sum(back) * Hkv * D * (1 + out) + 8 * Hkv * pages(back)
        return {"bytes": nbytes, "flops": 3 * T * case["rot"] * (Hq + Hkv) + 2 * T * Hkv * D}
    if case["kind"] == "read":
        return {"bytes": 2 * sum(lens) * Hkv * D * (1 + out) + 8 * Hkv * pages(lens), "flops": 2 * sum(lens) * Hkv * D}
    pairs = sum(n * (n_all - n) + n * (n + 1) // 2 for n_all, n in zip(lens, new))
    seen = [n_all for n_all, n in zip(lens, new) if n]
    return {"bytes": T * Hq * D * (el + out) + 2 * sum(seen) * Hkv * D + 8 * Hkv * pages(seen),
            "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------------ inputs


def _torch_dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _cu(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _turns(case):
    """Turns per position of each rotated pair, in 64 bits."""
    return [case["base"] ** (-2.0 * i / case["rot"]) / (2 * math.pi) for i in range(case["rot"] // 2)]


def _pages(g, pages, heads, ps, D):
    """Codes [pages, heads, ps, D] and scales [pages, heads] of values whose channels differ in size."""
    codes = torch.empty(pages, heads, ps, D, dtype=torch.uint8, device="cuda")
    scale = torch.empty(pages, heads, device="cuda")
    size = torch.exp(0.4 * torch.randn(1, heads, 1, D, device="cuda", generator=g))
    many = max(1, (1 << 26) // (heads * ps * D))
    for at in range(0, pages, many):
        to = min(pages, at + many)
        x = torch.randn(to - at, heads, ps, D, device="cuda", generator=g) * size
        s = x.abs().amax((2, 3)) / 127
        scale[at:to] = s
        codes[at:to] = (torch.round(x / s[:, :, None, None]) + 128).to(torch.uint8)
    return codes, scale


def _tiled(codes):
    """V codes [pages, heads, ps, D] in the order in which the cache holds them."""
    P, H, ps, D = codes.shape
    x = codes.view(P, H, ps // 32, 2, 4, 4, D // 32, 2, 16)  # tile, half, q, r, d / 32, e, c
    return x.permute(0, 1, 2, 6, 4, 8, 7, 3, 5).reshape(P, H, ps, D)


def _untiled(stored):
    """The reverse of ``_tiled``."""
    P, H, ps, D = stored.shape
    x = stored.view(P, H, ps // 32, D // 32, 4, 16, 2, 2, 4)  # tile, d / 32, q, c, e, half, r
    return x.permute(0, 1, 2, 7, 4, 8, 3, 6, 5).reshape(P, H, ps, D)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lens, new = _lens(case)
    B, Hq, Hkv, D, ps = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    dt = _torch_dtype(case["dtype"])
    widths = [-(-n // ps) for n in lens]
    max_pages = max(1, max(widths))
    total = sum(widths) + 3  # a pool has pages that no sequence holds
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(B, max_pages, dtype=torch.int32, device="cuda")
    held = torch.arange(max_pages, device="cuda")[None] < torch.tensor(widths, device="cuda")[:, None]
    table[held] = order[:sum(widths)]
    k, k_scale = _pages(g, total, Hkv, ps, D)
    v, v_scale = _pages(g, total, Hkv, ps, D)
    T = sum(new)
    st = {"case": case, "k": k, "v": _tiled(v), "k_scale": k_scale, "v_scale": v_scale, "table": table,
          "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu": _cu(new), "T": T,
          "max_new": max(new), "max_len": max(lens),
          "q": torch.randn(max(T, 1), Hq, D, device="cuda", generator=g).to(dt)[:T]}
    if case["kind"] == "append":
        st["k_new"] = torch.randn(T, Hkv, D, device="cuda", generator=g).to(dt)
        st["v_new"] = torch.randn(T, Hkv, D, device="cuda", generator=g).to(dt)
        st["turns"] = torch.tensor(_turns(case), dtype=torch.float64, device="cuda")
        # the same as 0.64 fixed point, which a position multiplies without rounding
        st["freqs"] = torch.tensor([round(f * 2**64) for f in _turns(case)], dtype=torch.int64, device="cuda")
        back = _touched(case)
        st["cu_back"], st["T_back"], st["max_back"] = _cu(back), sum(back), max(back)
        # the touched pages as a scheduler lists them: (sequence, page, its tokens that are new)
        slots = [(b, j) for b in range(B) if new[b] for j in range((lens[b] - new[b]) // ps, -(-lens[b] // ps))]
        at = torch.tensor(slots, dtype=torch.int64, device="cuda").reshape(-1, 2)
        first = st["lens"].long() - torch.tensor(new, device="cuda")  # position of a sequence's first new token
        pos = at[:, 1:] * ps + torch.arange(ps, device="cuda")[None]
        b = at[:, 0]
        st["slot_page"] = table[b, at[:, 1]].long()
        st["slot_token"] = torch.where((pos >= first[b, None]) & (pos < st["lens"][b, None]),
                                       pos - first[b, None] + st["cu"][b, None], torch.full_like(pos, -1))
        st["slot_old"] = at[:, 1] * ps < first[b]
    if case["kind"] == "read":
        st["cu_back"], st["T_back"], st["max_back"] = _cu(lens), sum(lens), max(lens)
    return st


# -------------------------------------------------------------- plain form


def _tokens(st, cu, T):
    """Sequence and position of each of T packed tokens, the last ones of each sequence."""
    n = torch.arange(T, device="cuda")
    b = torch.searchsorted(cu[1:].long(), n, right=True)
    return b, n - cu[b].long() + st["lens"][b].long() - (cu[b + 1] - cu[b]).long()


def _rotated(x, pos, st):
    """x [T, H, D] with its first rot elements rotated by position; angles in 64 bits."""
    case = st["case"]
    rot = case["rot"]
    t = pos[:, None].double() * st["turns"][None]
    a = (t - torch.round(t)) * (2 * math.pi)
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    x = x.float()
    y = x.clone()
    if case["interleaved"]:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = x0 * c - x1 * s, x1 * c + x0 * s
    else:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def _merge(st, codes, scale, rows):
    """The touched pages' codes [slots, H, ps, D] with the new rows in them, and their scales."""
    tok, page = st["slot_token"], st["slot_page"]
    new = (tok >= 0)[:, None, :, None]
    x = rows[tok.clamp(min=0)].permute(0, 2, 1, 3) * new  # [slots, H, ps, D]
    old = torch.where(st["slot_old"][:, None], scale[page], torch.zeros_like(scale[page]))
    s = torch.maximum(old, (x.abs().amax((2, 3)) / 127).clamp(min=2.0**-126))
    kept = torch.round((codes.float() - 128) * (old / s)[:, :, None, None])
    kept = torch.where((old == s)[:, :, None, None], codes.float() - 128, kept)
    made = torch.where(new, torch.round(x / s[:, :, None, None]), kept)
    live = new | st["slot_old"][:, None, None, None]
    return torch.where(live, made + 128, codes.float()).to(torch.uint8), s


def _plain_append(st):
    _, pos = _tokens(st, st["cu"], st["T"])
    q = _rotated(st["q"], pos, st).to(st["q"].dtype)
    page = st["slot_page"]
    k, s = _merge(st, st["k"][page], st["k_scale"], _rotated(st["k_new"], pos, st))
    st["k"][page], st["k_scale"][page] = k, s
    v, s = _merge(st, _untiled(st["v"][page]), st["v_scale"], st["v_new"].float())
    st["v"][page], st["v_scale"][page] = _tiled(v), s
    return q


def _plain_read(st):
    ps = st["case"]["page"]
    b, pos = _tokens(st, st["cu_back"], st["T_back"])
    page, row = st["table"][b, pos // ps].long(), pos % ps
    dt = _torch_dtype(st["case"]["out"])
    k = (st["k"][page, :, row].float() - 128) * st["k_scale"][page][:, :, None]
    t, D = row % 32, st["case"]["D"]
    v = st["v"].view(*st["v"].shape[:2], ps // 32, D // 32, 4, 16, 2, 2, 4)
    v = v[page, :, row // 32, :, t // 4 % 4, :, :, t // 16, t % 4]  # [T, H, D / 32, c, e]
    v = v.transpose(3, 4).reshape(len(b), -1, D)
    v = (v.float() - 128) * st["v_scale"][page][:, :, None]
    return k.to(dt), v.to(dt)


def _dense(st):
    """K and V [B, Hkv, max_len, D] in 32 bits; what no sequence holds is whatever its page has."""
    t = st["table"].long()
    B, M = t.shape
    P, H, ps, D = st["k"].shape
    k = (st["k"][t].float() - 128) * st["k_scale"][t][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, H, M * ps, D)[:, :, :st["max_len"]]
    v = _untiled(st["v"][t].view(B * M, H, ps, D)).view(B, M, H, ps, D)
    v = (v.float() - 128) * st["v_scale"][t][..., None, None]
    return k, v.permute(0, 2, 1, 3, 4).reshape(B, H, M * ps, D)[:, :, :st["max_len"]]


def _plain_attention(st):
    case = st["case"]
    B, Hq, Hkv, D, N = case["B"], case["Hq"], case["Hkv"], case["D"], st["max_new"]
    G = Hq // Hkv
    k, v = _dense(st)
    cu, lens = st["cu"].long(), st["lens"].long()
    n_new = cu[1:] - cu[:-1]
    i = torch.arange(N, device="cuda")
    row = (cu[:-1, None] + i[None]).clamp(max=st["T"] - 1)
    q = st["q"].float()[row] * D**-0.5  # [B, N, Hq, D], rows past a sequence's own unused
    q = q.view(B, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hkv, N, G, -1)
    last = (lens - n_new)[:, None] + i[None]  # the last key that a row sees
    keep = torch.arange(st["max_len"], device="cuda")[None, None] <= last[:, :, None]
    s = s.masked_fill(~keep[:, None, :, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, N * G, -1), v).view(B, Hkv, N, G, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq, D)
    b, pos = _tokens(st, st["cu"], st["T"])
    return o[b, pos - (lens - n_new)[b]].to(_torch_dtype(case["out"]))


# ------------------------------------------------------------------- passes


def _handles(st):
    """The cache and batch handles that a user's program keeps beside its tensors."""
    if "cache" not in st:
        from hipgpt_amd import kvcache

        c = st["case"]
        st["cache"] = kvcache.CacheQ8(st["k"], st["v"], st["k_scale"], st["v_scale"])
        decode = c["new_lo"] == c["new_hi"] == 1
        st["batch"] = kvcache.Batch(st["table"], st["lens"], None if decode else st["cu"], max_new=st["max_new"],
                                    max_len=st["max_len"])
        if "cu_back" in st:
            st["back"] = kvcache.Batch(st["table"], st["lens"], st["cu_back"], max_new=st["max_back"],
                                       max_len=st["max_len"])
    return st["cache"], st["batch"]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from hipgpt_amd import kvcache

        cache, batch = _handles(state)
        dt = _torch_dtype(case["out"])
        if kind == "append":
            q = kvcache.append(cache, batch, state["q"], state["k_new"], state["v_new"], freqs=state["freqs"],
                               interleaved=case["interleaved"])
            k, v = kvcache.read(cache, state["back"], state["T_back"], dtype=dt)
            return {"q": q, "k": k, "v": v, "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        if kind == "read":
            k, v = kvcache.read(cache, state["back"], state["T_back"], dtype=dt)
            return {"k": k, "v": v}
        if kind == "decode":
            return kvcache.decode(cache, batch, state["q"], out_dtype=dt)
        return kvcache.prefill(cache, batch, state["q"], out_dtype=dt)
    if kind == "append":
        q = _plain_append(state)
        k, v = _plain_read(state)
        return {"q": q, "k": k, "v": v, "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if kind == "read":
        k, v = _plain_read(state)
        return {"k": k, "v": v}
    return _plain_attention(state)


# -------------------------------------------------------------- 64-bit form


def _exact_rows(st, which, b, n):
    """The first n tokens of sequence b as [H, n, D] in 64 bits."""
    ps = st["case"]["page"]
    pages = st["table"][b, :-(-n // ps)].long()
    codes = st["k"][pages] if which == "k" else _untiled(st["v"][pages])
    x = (codes.double() - 128) * st[which + "_scale"][pages].double()[:, :, None, None]
    return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def _exact_rotation(x, pos, case):
    """x [n, H, D] at positions pos, pair by pair as complex numbers."""
    rot = case["rot"]
    f = torch.tensor(_turns(case), dtype=torch.float64, device="cuda")
    w = torch.polar(torch.ones(len(pos), 1, len(f), dtype=torch.float64, device="cuda"),
                    (2 * math.pi * torch.remainder(pos.double()[:, None] * f, 1.0))[:, None])
    y = x.double().clone()
    lead = y[..., :rot]
    pairs = lead.unflatten(-1, (-1, 2)) if case["interleaved"] else lead.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    y[..., :rot] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return y


def _exact_append(st):
    case, (lens, new) = st["case"], _lens(st["case"])
    ps, H, D = case["page"], case["Hkv"], case["D"]
    scales = {"k": st["k_scale"].double(), "v": st["v_scale"].double()}
    q, back, at = [], {"k": [], "v": []}, 0
    for b, (n_all, n) in enumerate(zip(lens, new)):
        if not n:
            continue
        pos = torch.arange(n_all - n, n_all, device="cuda")
        q.append(_exact_rotation(st["q"][at:at + n], pos, case))
        rows = {"k": _exact_rotation(st["k_new"][at:at + n], pos, case), "v": st["v_new"][at:at + n].double()}
        at += n
        from_ = (n_all - n) // ps * ps
        for which in ("k", "v"):
            old = _exact_rows(st, which, b, n_all - n)[:, from_:]
            all_ = torch.cat([old, rows[which].transpose(0, 1)], 1)
            n_old, pages = old.shape[1], -(-all_.shape[1] // ps)
            full = torch.zeros(H, pages * ps, D, dtype=torch.float64, device="cuda")
            full[:, :all_.shape[1]] = all_
            fresh = full.clone()
            fresh[:, :n_old] = 0
            ids = st["table"][b, from_ // ps:from_ // ps + pages].long()
            s = (fresh.view(H, pages, -1).abs().amax(-1) / 127).clamp(min=2.0**-126)
            if n_old:
                s[:, 0] = torch.maximum(s[:, 0], scales[which][ids[0]])
            scales[which][ids] = s.t()
            step = s.repeat_interleave(ps, 1)[:, :, None]
            back[which].append((torch.round(full / step) * step)[:, :all_.shape[1]].transpose(0, 1))
    return {"q": torch.cat(q), "k": torch.cat(back["k"]), "v": torch.cat(back["v"]), "k_scale": scales["k"],
            "v_scale": scales["v"]}


def exact(case, seed):
    st = prepare(case, seed)
    lens, new = _lens(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "read":
        return {w: torch.cat([_exact_rows(st, w, b, n).transpose(0, 1) for b, n in enumerate(lens)]) for w in ("k", "v")}
    outs, at = [], 0
    for b, (n_all, n) in enumerate(zip(lens, new)):
        if not n:
            continue
        k, v = _exact_rows(st, "k", b, n_all), _exact_rows(st, "v", b, n_all)
        seen = torch.ones(n, n_all, dtype=torch.bool, device="cuda").tril(n_all - n)
        q = st["q"][at:at + n].double()
        at += n
        heads = []
        for h in range(Hq):
            s = q[:, h] @ k[h * Hkv // Hq].t() / math.sqrt(D)
            s[~seen] = -math.inf
            heads.append(torch.softmax(s, -1) @ v[h * Hkv // Hq])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
