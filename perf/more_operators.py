"""Performance cases of rotary positions, their way into the paged cache, and
attention over a latent cache.

A case's "kind" says which operator it stands for:

- "rotate" and "tables": rotary positions of query or key rows as a projection
  leaves them (rope_rows), with adjacent pairs or halves of the head, over all
  of it or a part; and the cosine and sine tables of a context length, scaled
  for contexts longer than the trained one (rope_tables).
- "append" and "latent_append": a step's new rows on their way into the pages:
  queries and keys rotated, keys and values rounded to the page type and put at
  their slots, in one call (rope_append); the same for a latent cache, whose
  pages hold one shared vector a token, a latent part and a rotated part
  (latent_append).
- "latent": attention of a step's queries over the pages of a latent cache, in
  the absorbed form: every head's key is the token's whole row and its value the
  row's latent part (paged_latent_attention).
- "expanded": the same attention in its expanded form, for prompts: each head
  has keys and values of its own, and a part of every key is shared by the heads
  (latent_prefill_attention).

With `own` false the operators run in their plain forms, with it true through
the framework's entry points.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
P = 16       # tokens of a page
ROPE = 64    # rotated part of a latent cache's row
NOPE = 128   # per-head key part without position, and value size, of the expanded form
K_SCALE, V_SCALE = 0.03, 0.015  # fp8 scales of a calibrated cache
BASE = 500000.0


# ------------------------------------------------------------------ cases ----
def listed():
    return [
        # One chat's queries of one layer: launch and call.
        dict(name="rotate_one", kind="rotate", tokens=1, heads=32, dim=128, rotary=128,
             layout="halves", fused=True, rows=8192),
        # Prompts packed side by side, half of a 96-wide head rotated.
        dict(name="rotate_part", kind="rotate", tokens=8191, heads=40, dim=96, rotary=48,
             layout="pairs", fused=True, rows=131072),
        # Tables for 131072 positions of a model trained on 8192.
        dict(name="tables_long", kind="tables", rows=131072, rotary=128, scaling="ramp",
             factor=16.0, original=8192),
        # One chat's token of one layer, 32/8 heads, bf16 pages.
        dict(name="append_one", kind="append", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128,
             rotary=128, layout="halves", ragged=False, dtype="bf16"),
        # A chunked prefill step: 16 sequences of 512 rows, fp32 pages.
        dict(name="append_chunk", kind="append", batch=16, tokens=512, q_heads=32, kv_heads=8,
             dim=128, rotary=128, layout="halves", ragged=False, dtype="f32"),
        # Ragged chunks into a latent cache with fp8 pages, 128 heads' queries.
        dict(name="append_latent", kind="latent_append", batch=33, tokens=65, q_heads=128,
             latent=512, layout="pairs", ragged=True, dtype="fp8"),
        # One chat at its beginning, fp32 pages: launches and latency.
        dict(name="latent_one", kind="latent", batch=1, tokens=1, q_heads=16, latent=512, low=121,
             high=121, ragged=False, dtype="f32"),
        # One chat over a very long context, three tokens a step.
        dict(name="latent_long", kind="latent", batch=1, tokens=3, q_heads=16, latent=512,
             low=131071, high=131071, ragged=False, dtype="bf16"),
        # A full server: 64 sequences, contexts log-uniform in [512, 8192]; one
        # GPU's 16 heads of a model split over eight (fp8 pages: the pages are
        # what it takes), and all 128 heads (bf16 pages: the arithmetic is).
        dict(name="latent_shard", kind="latent", batch=64, tokens=1, q_heads=16, latent=512,
             low=512, high=8192, ragged=False, dtype="fp8"),
        dict(name="latent_server", kind="latent", batch=64, tokens=1, q_heads=128, latent=512,
             low=512, high=8192, ragged=False, dtype="bf16"),
        # Short prompts of a batch, each with its own length.
        dict(name="expand_ragged", kind="expanded", batch=5, heads=20, tokens=257, keys=257,
             ragged=True),
        # A prompt's last chunk over what lies before it: the most arithmetic.
        dict(name="expand_chunk", kind="expanded", batch=4, heads=32, tokens=512, keys=4096,
             ragged=False),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotate", "tables", "append", "append", "latent_append", "latent", "latent",
                       "latent", "expanded", "expanded"])
    layout = rng.choice(["pairs", "halves"])
    dtype = rng.choice(["f32", "bf16", "fp8"])
    ragged = rng.random() < 0.4
    if kind == "rotate":
        heads, dim = _log_int(rng, 1, 64), rng.choice([40, 64, 80, 96, 128, 192, 256])
        return dict(kind=kind, tokens=_log_int(rng, 1, min(8191, 31000000 // (heads * dim))),
                    heads=heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2, 2, 32, 18]),
                    layout=layout, fused=rng.random() < 0.6, rows=_log_int(rng, 64, 131072))
    if kind == "tables":
        return dict(kind=kind, rows=_log_int(rng, 1, 131072),
                    rotary=rng.choice([16, 50, 64, 96, 128]),
                    scaling=rng.choice(["none", "linear", "ntk", "ramp", "bands"]),
                    factor=rng.choice([1.0, 2.5, 4.0, 8.0, 16.0]),
                    original=rng.choice([2048, 4096, 8192]))
    batch = _log_int(rng, 1, 64)
    if kind == "append":
        kv_heads, group = rng.choice([(8, 4), (8, 4), (8, 1), (32, 1), (4, 8), (3, 5), (1, 16)])
        dim = rng.choice([128, 128, 128, 64, 80])
        return dict(kind=kind, batch=batch, tokens=_log_int(rng, 1, min(512, 4096 // batch)),
                    q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2]), layout=layout, ragged=ragged,
                    dtype=dtype)
    latent = rng.choice([512, 512, 512, 256])
    if kind == "latent_append":
        return dict(kind=kind, batch=batch, tokens=_log_int(rng, 1, min(512, 2145 // batch)),
                    q_heads=rng.choice([1, 5, 16, 40, 128]), latent=latent, layout=layout,
                    ragged=ragged, dtype=dtype)
    if kind == "latent":
        q_heads = rng.choice([8, 16, 16, 20, 40, 64, 128, 128])
        tokens = rng.choice([1, 1, 1, 2, 3, _log_int(rng, 1, 64)])
        most = 20000000 // (q_heads * tokens * batch)  # tokens of the longest: less work than listed
        high = _log_int(rng, 1, max(1, min(8192, most)))
        if batch <= 2 and rng.random() < 0.5:
            high = min(most, _log_int(rng, 8192, 131071))
        return dict(kind=kind, batch=batch, tokens=tokens, q_heads=q_heads, latent=latent,
                    low=rng.choice([high, high // 4, high // 16, 0]), high=high, ragged=ragged,
                    dtype=dtype)
    heads = rng.choice([1, 5, 12, 20, 32])
    tokens = _log_int(rng, 1, 1024)
    batch = min(batch, max(1, 65536 // (heads * tokens)))
    keys = _log_int(rng, tokens, max(tokens, min(8192, 250000000 // (batch * heads * tokens))))
    if batch * heads * tokens * keys > 250000000 or rng.random() < 0.4:
        keys = tokens
    return dict(kind=kind, batch=batch, heads=heads, tokens=tokens, keys=keys, ragged=ragged)


# ----------------------------------------------------------------- inputs ----
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 31)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _case_rng(case, salt):
    return np.random.default_rng([salt, case["batch"], case["tokens"], case.get("high", 0),
                                  case.get("keys", 0), case.get("q_heads", 0)])


def _counts(case):
    """New tokens of each sequence (part of the case)."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * b
    return [int(x) for x in _case_rng(case, 2).integers(min(1, t // 2), t + 1, size=b)]


def _lengths(case):
    """Tokens in the pages of each sequence, the new ones among them (part of
    the case)."""
    low, high, n = case["low"], case["high"], case["batch"]
    rng = _case_rng(case, 1)
    if low > 0 and high > 4 * low:  # contexts of a batch spread over their logarithm
        v = np.exp(rng.uniform(math.log(low), math.log(high + 1), size=n)).astype(np.int64)
        v = [int(min(high, max(low, x))) for x in v]
    else:
        v = [int(x) for x in rng.integers(min(low, high), high + 1, size=n)]
    return [max(x, c) for x, c in zip(v, _counts(case))]


def _key_counts(case):
    """Keys of each sequence of an expanded case, its new tokens the last ones."""
    counts, s, t = _counts(case), case["keys"], case["tokens"]
    if not case["ragged"]:
        return [s] * len(counts)
    before = _case_rng(case, 3).integers(0, s - t + 1, size=len(counts))
    return [int(n) + c for n, c in zip(before, counts)]


def _i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=DEV)


def _angles(rows, rotary):
    """Cosines and sines [rows, rotary / 2] of an unscaled model."""
    i = torch.arange(rotary // 2, device=DEV, dtype=torch.float64)
    a = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * BASE ** (-2.0 * i / rotary)
    return torch.cos(a).float(), torch.sin(a).float()


def _pool(g, dtype, scale, channel, *shape):
    """Pages of random rows in their element type."""
    x = _randn(g, *shape)
    if channel is not None:
        x *= channel
    if dtype == "bf16":
        return x.to(torch.bfloat16)
    if dtype == "fp8":
        return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return x


def _slots(case, seed, counts):
    """Slots [batch, tokens] of the new tokens behind histories that end
    anywhere in a page (-1 behind a sequence's tokens), the position of each
    sequence's first one, and the number of pages."""
    b, t = case["batch"], case["tokens"]
    each = (t + 2 * P - 2) // P
    physical = b * each + 2
    rng = np.random.default_rng(int(seed) + 6)
    order = rng.permutation(physical)
    starts = rng.integers(0, 4096, size=b)
    at = starts[:, None] % P + np.arange(t)
    slots = order[np.arange(b)[:, None] * each + at // P].astype(np.int64) * P + at % P
    slots[np.arange(t)[None] >= np.asarray(counts)[:, None]] = -1
    return slots, starts, physical


def _rotate_inputs(case, seed):
    g = _generator(seed)
    n, h, d = case["tokens"], case["heads"], case["dim"]
    # The rows lie among a projection's other outputs, or by themselves.
    x = _randn(g, n, h + 16 if case["fused"] else h, d)[:, :h]
    positions = torch.randint(case["rows"], (n,), device=DEV, generator=g, dtype=torch.int32)
    cos, sin = _angles(case["rows"], case["rotary"])
    return dict(x=x, positions=positions, cos=cos, sin=sin)


def _append_inputs(case, seed):
    g = _generator(seed)
    b, t, d = case["batch"], case["tokens"], case["dim"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    counts = _counts(case)
    slots, starts, physical = _slots(case, seed, counts)
    kp = _pool(g, case["dtype"], K_SCALE, None, physical, hkv, P, d)
    vp = _pool(g, case["dtype"], V_SCALE, None, physical, hkv, P, d)
    # One projection's output: queries, keys and values of a token side by side.
    rows = _randn(g, b, t, hq + 2 * hkv, d).transpose(1, 2)
    cos, sin = _angles(4096 + t, case["rotary"])
    return dict(q=rows[:, :hq], k=rows[:, hq:hq + hkv], v=rows[:, hq + hkv:], kp=kp, vp=vp,
                slots=torch.as_tensor(slots, device=DEV), starts=_i32(starts), cos=cos, sin=sin,
                counts=counts)


def _latent_append_inputs(case, seed):
    g = _generator(seed)
    b, t, hq, n = case["batch"], case["tokens"], case["q_heads"], case["latent"]
    counts = _counts(case)
    slots, starts, physical = _slots(case, seed, counts)
    pool = _pool(g, case["dtype"], K_SCALE, None, physical, P, n + ROPE)
    cos, sin = _angles(4096 + t, ROPE)
    # The rotated parts come out of projections beside the parts without position.
    q = _randn(g, b, t, hq, NOPE + ROPE).transpose(1, 2)[..., NOPE:]
    down = _randn(g, b, t, n + ROPE)
    return dict(q=q, latent=_randn(g, b, t, n), rope_key=down[..., n:], pool=pool,
                slots=torch.as_tensor(slots, device=DEV), starts=_i32(starts), cos=cos, sin=sin,
                counts=counts)


def _latent_inputs(case, seed):
    g = _generator(seed)
    b, t, hq, n = case["batch"], case["tokens"], case["q_heads"], case["latent"]
    lengths = _lengths(case)
    pages = [(x + P - 1) // P for x in lengths]
    physical = sum(pages) + 3
    channel = torch.exp(0.4 * _randn(g, n + ROPE))  # elements differ in size by channel
    pool = _pool(g, case["dtype"], K_SCALE, channel, physical, P, n + ROPE)
    order = np.random.default_rng(int(seed) + 5).permutation(physical)
    tables = np.zeros((b, max(1, max(pages))), np.int32)
    at = 0
    for i, m in enumerate(pages):
        tables[i, :m] = order[at:at + m]
        at += m
    return dict(q=_randn(g, b, hq, t, n + ROPE), pool=pool, tables=_i32(tables),
                lengths=_i32(lengths), host_lengths=lengths, counts=_counts(case))


def _expanded_inputs(case, seed):
    g = _generator(seed)
    b, h, t, s = case["batch"], case["heads"], case["tokens"], case["keys"]
    # Queries and expanded keys and values as their projections leave them.
    q = _randn(g, b, t, h, NOPE + ROPE).transpose(1, 2)
    kv = _randn(g, b, s, h, 2 * NOPE).transpose(1, 2)
    return dict(q=q, k=kv[..., :NOPE], v=kv[..., NOPE:], rope_key=_randn(g, b, s, ROPE),
                counts=_counts(case), key_counts=_key_counts(case))


def _inputs(case, seed):
    return {"rotate": _rotate_inputs, "append": _append_inputs, "latent": _latent_inputs,
            "latent_append": _latent_append_inputs, "expanded": _expanded_inputs}[case["kind"]](
                case, seed)


def _softmax_scale(case):
    return 1.0 / math.sqrt(NOPE + ROPE)


def prepare(case, seed):
    if case["kind"] == "tables":
        shape = (case["rows"], case["rotary"] // 2)
        # (Another seed's sequence starts elsewhere.)
        return dict(case, cos=torch.empty(shape, device=DEV), sin=torch.empty(shape, device=DEV),
                    first=int(seed) % 1000)
    s = _inputs(case, seed)
    s.update((k, case[k]) for k in ("kind", "layout", "rotary", "dtype") if k in case)
    if "counts" in s:
        b, t = case["batch"], case["tokens"]
        s["token_counts"] = _i32(s["counts"]) if case["ragged"] else None
        # Which of the rows are a sequence's, as the server that laid them out knows.
        live = torch.arange(t, device=DEV)[None] < _i32(s["counts"])[:, None]
        s["live"] = live.flatten().nonzero()[:, 0]
        s["at"] = torch.arange(t, device=DEV)[None] - _i32(s["counts"])[:, None]
    if case["kind"] == "rotate":
        s["out"] = torch.empty(s["x"].shape, device=DEV)
    elif case["kind"] == "append":
        s["q_out"], s["k_out"], s["v_out"] = (torch.zeros(s[x].shape, device=DEV) for x in "qkv")
    elif case["kind"] == "latent_append":
        # The absorbed queries' buffer, whose last part the rotated ones fill.
        whole = torch.zeros(*s["q"].shape[:3], case["latent"] + ROPE, device=DEV)
        s["q_out"] = whole[..., case["latent"]:]
    elif case["kind"] == "latent":
        s["out"] = torch.zeros(*s["q"].shape[:3], case["latent"], device=DEV)
        s["scale"] = _softmax_scale(case)
        if own:
            import helix_runtime_amd as hx
            s["workspace"] = hx.latent_workspace(case["batch"], case["q_heads"], case["tokens"],
                                                 case["latent"])
    elif case["kind"] == "expanded":
        s["out"] = torch.zeros(*s["q"].shape[:3], NOPE, device=DEV)
        s["scale"] = _softmax_scale(case)
        s["key_lengths"] = _i32(s["key_counts"]) if case["ragged"] else None
        s["ends"] = _i32(s["key_counts"])
        if own:
            import helix_runtime_amd as hx
            s["workspace"] = hx.latent_prefill_workspace(case["batch"], case["heads"],
                                                         case["tokens"], case["keys"])
    return s


# -------------------------------------------------------------------- run ----
def run(s):
    if own:
        return _OWN[s["kind"]](s)
    return _PLAIN[s["kind"]](s)


def _rotate_own(s):
    import helix_runtime_amd as hx
    hx.rope_rows(s["x"], s["cos"], s["sin"], s["out"], positions=s["positions"],
                 layout=s["layout"], rotary_dim=s["rotary"])
    return s["out"]


def _tables_own(s):
    import helix_runtime_amd as hx
    hx.rope_tables(s["cos"], s["sin"], base=BASE, first_position=s["first"], scaling=s["scaling"],
                   factor=s["factor"], original_length=s["original"])
    return {"cos": s["cos"], "sin": s["sin"]}


def _append_own(s):
    import helix_runtime_amd as hx
    hx.rope_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["starts"], s["slots"], s["cos"],
                   s["sin"], s["q_out"], key_out=s["k_out"], value_out=s["v_out"],
                   layout=s["layout"], rotary_dim=s["rotary"], token_counts=s["token_counts"],
                   page_dtype=s["dtype"], k_scale=K_SCALE, v_scale=V_SCALE)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "keys": _pages(s, s["kp"]),
            "values": _pages(s, s["vp"])}


def _latent_append_own(s):
    import helix_runtime_amd as hx
    hx.latent_append(s["latent"], s["rope_key"], s["pool"], s["starts"], s["slots"], s["cos"],
                     s["sin"], query=s["q"], query_out=s["q_out"], layout=s["layout"],
                     token_counts=s["token_counts"], page_dtype=s["dtype"], page_scale=K_SCALE)
    return {"q": s["q_out"], "pages": _pages(s, s["pool"])}


def _latent_own(s):
    import helix_runtime_amd as hx
    hx.paged_latent_attention(s["q"], s["pool"], s["tables"], s["lengths"], s["out"],
                              s["workspace"], s["scale"], token_counts=s["token_counts"],
                              page_dtype=s["dtype"], page_scale=K_SCALE)
    return s["out"]


def _expanded_own(s):
    import helix_runtime_amd as hx
    hx.latent_prefill_attention(s["q"], s["k"], s["rope_key"], s["v"], s["out"], s["workspace"],
                                s["scale"], key_lengths=s["key_lengths"],
                                token_counts=s["token_counts"])
    return s["out"]


def _pages(s, pool):
    """Pages as the numbers they hold (fp8: to be multiplied by the cache's
    scale, a constant)."""
    return pool.view(torch.float8_e4m3fn) if s["dtype"] == "fp8" else pool


def _widened(s, pool, scale):
    if s["dtype"] == "fp8":
        return pool.view(torch.float8_e4m3fn).to(torch.float32) * scale
    return pool.to(torch.float32)


def _rotated(s, x, cos, sin, rotary):
    """Rows [..., dim] with their first `rotary` elements rotated."""
    if s["layout"] == "pairs":
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return y if rotary == x.shape[-1] else torch.cat([y, x[..., rotary:]], dim=-1)


def _rotate(s):
    at = s["positions"].long()
    s["out"].copy_(_rotated(s, s["x"], s["cos"][at][:, None], s["sin"][at][:, None], s["rotary"]))
    return s["out"]


def _tables(s):
    d, kind, factor, trained = s["rotary"], s["scaling"], s["factor"], s["original"]
    i = torch.arange(d // 2, device=DEV, dtype=torch.float64)
    base = BASE * factor ** (d / (d - 2)) if kind == "ntk" else BASE
    f = base ** (-2.0 * i / d)
    if kind == "linear":
        f = f / factor
    elif kind == "ramp":  # from as they are to divided, between 32 and 1 turns over `trained`
        low = max(math.floor(d * math.log(trained / (32 * 2 * math.pi)) / (2 * math.log(BASE))), 0)
        high = min(math.ceil(d * math.log(trained / (2 * math.pi)) / (2 * math.log(BASE))), d - 1)
        part = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * part + f * (1 - part)
    elif kind == "bands":  # the same by wavelength, between 4 turns and 1
        turns = trained * f / (2 * math.pi)
        part = ((turns - 1) / 3).clamp(0, 1)
        f = f / factor * (1 - part) + f * part
    at = torch.arange(s["first"], s["first"] + s["rows"], device=DEV, dtype=torch.float64)
    a = at[:, None] * f
    s["cos"].copy_(torch.cos(a))
    s["sin"].copy_(torch.sin(a))
    return {"cos": s["cos"], "sin": s["sin"]}


def _put_live(s, out, x):
    """Rows [batch, heads, tokens, ..] of the sequences' own tokens; the others stay."""
    t = x.shape[2]
    b, at = s["live"] // t, s["live"] % t
    out[b, :, at] = x[b, :, at]


def _on_pages(s, x, scale):
    """fp32 rows as elements of a page."""
    if s["dtype"] == "bf16":
        return x.to(torch.bfloat16)
    if s["dtype"] == "fp8":
        by = torch.full((), scale, device=x.device)  # a tensor: a true fp32 division
        return (x / by).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return x


def _step_angles(s):
    at = (s["starts"][:, None] + torch.arange(s["slots"].shape[1], device=DEV)).long()
    return s["cos"][at], s["sin"][at]  # [batch, tokens, rotary / 2]


def _append(s):
    cos, sin = _step_angles(s)
    t = s["slots"].shape[1]
    q = _rotated(s, s["q"], cos[:, None], sin[:, None], s["rotary"])
    k = _rotated(s, s["k"], cos[:, None], sin[:, None], s["rotary"])
    _put_live(s, s["q_out"], q)
    _put_live(s, s["k_out"], k)
    _put_live(s, s["v_out"], s["v"])
    b, at = s["live"] // t, s["live"] % t
    slot = s["slots"].flatten()[s["live"]]
    s["kp"][slot // P, :, slot % P] = _on_pages(s, k[b, :, at], K_SCALE)
    s["vp"][slot // P, :, slot % P] = _on_pages(s, s["v"][b, :, at], V_SCALE)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "keys": _pages(s, s["kp"]),
            "values": _pages(s, s["vp"])}


def _latent_append(s):
    cos, sin = _step_angles(s)
    _put_live(s, s["q_out"], _rotated(s, s["q"], cos[:, None], sin[:, None], ROPE))
    row = torch.cat([s["latent"], _rotated(s, s["rope_key"], cos, sin, ROPE)], dim=-1)
    slot = s["slots"].flatten()[s["live"]]
    s["pool"][slot // P, slot % P] = _on_pages(s, row.flatten(0, 1)[s["live"]], K_SCALE)
    return {"q": s["q_out"], "pages": _pages(s, s["pool"])}


def _softmax_rows(x, seen, v):
    """exp(x - max) v / sum over the keys that `seen` leaves, 0 where it leaves none."""
    x = x.masked_fill_(~seen, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    x = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = x.sum(dim=-1, keepdim=True)
    return torch.matmul(x, v) / torch.where(total > 0, total, 1.0)


def _latent(s):
    b, hq, t, w = s["q"].shape
    n = w - ROPE
    rows = _widened(s, s["pool"][s["tables"].long()], K_SCALE).flatten(1, 2)  # [b, keys, w]
    x = torch.matmul(s["q"].reshape(b, hq * t, w), rows.transpose(1, 2)) * s["scale"]
    ends = s["lengths"][:, None] + s["at"] + 1  # [b, t]
    seen = torch.arange(rows.shape[1], device=DEV) < ends[:, :, None]
    y = _softmax_rows(x, seen.repeat(1, hq, 1), rows[..., :n])
    _put_live(s, s["out"], y.view(b, hq, t, n))
    return s["out"]


def _expanded(s):
    b, h, n = s["k"].shape[:3]
    k = torch.cat([s["k"], s["rope_key"][:, None].expand(b, h, n, ROPE)], dim=-1)
    x = torch.matmul(s["q"], k.transpose(2, 3)) * s["scale"]
    ends = s["ends"][:, None] + s["at"] + 1
    seen = torch.arange(n, device=DEV) < ends[:, None, :, None]
    _put_live(s, s["out"], _softmax_rows(x, seen, s["v"]))
    return s["out"]


_PLAIN = {"rotate": _rotate, "tables": _tables, "append": _append, "latent": _latent,
          "latent_append": _latent_append, "expanded": _expanded}
_OWN = {"rotate": _rotate_own, "tables": _tables_own, "append": _append_own,
        "latent": _latent_own, "latent_append": _latent_append_own, "expanded": _expanded_own}


# ------------------------------------------------------------------- work ----
def work(case):
    kind = case["kind"]
    if kind == "tables":
        return {"bytes": 4 * case["rows"] * case["rotary"], "flops": 3 * case["rows"] * case["rotary"]}
    if kind == "rotate":
        n, h = case["tokens"], case["heads"]
        # (Table rows that several tokens use are read once.)
        table = 4 * min(n, case["rows"]) * case["rotary"]
        return {"bytes": 8 * n * h * case["dim"] + table + 4 * n, "flops": 3 * n * h * case["rotary"]}
    counts = _counts(case)
    n = sum(counts)
    size = {"f32": 4, "bf16": 2, "fp8": 1}.get(case.get("dtype"), 4)
    if kind == "append":
        hq, hkv, d, r = case["q_heads"], case["kv_heads"], case["dim"], case["rotary"]
        return {"bytes": n * (8 * (hq + 2 * hkv) * d + 2 * size * hkv * d + 4 * r + 12),
                "flops": 3 * n * (hq + hkv) * r}
    if kind == "latent_append":
        hq, w = case["q_heads"], case["latent"] + ROPE
        return {"bytes": n * (8 * hq * ROPE + (4 + size) * w + 4 * ROPE + 12),
                "flops": 3 * n * (hq + 1) * ROPE}
    if kind == "latent":
        hq, w = case["q_heads"], case["latent"] + ROPE
        lengths = _lengths(case)
        pairs = sum(c * (x - (c - 1) / 2) for x, c in zip(lengths, counts))
        return {"bytes": size * w * sum(lengths) + 4 * hq * n * (w + case["latent"]),
                "flops": int(2 * hq * (w + case["latent"]) * pairs)}
    h, keys = case["heads"], _key_counts(case)
    pairs = sum(c * (x - (c - 1) / 2) for x, c in zip(keys, counts))
    return {"bytes": 4 * (sum(keys) * (2 * h * NOPE + ROPE) + n * h * (2 * NOPE + ROPE)),
            "flops": int(2 * h * (2 * NOPE + ROPE) * pairs)}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return _exact_tables(case, seed)
    s = _inputs(case, seed)
    if kind == "rotate":
        at = s["positions"].cpu().numpy()
        return torch.from_numpy(_turn(case["layout"], s["x"].cpu().numpy().astype(np.float64),
                                      s["cos"].cpu().numpy()[at][:, None],
                                      s["sin"].cpu().numpy()[at][:, None], case["rotary"]))
    if kind == "append":
        return _exact_append(case, s)
    if kind == "latent_append":
        return _exact_latent_append(case, s)
    if kind == "latent":
        return _exact_latent(case, s)
    return _exact_expanded(case, s)


def _exact_tables(case, seed):
    d, kind, factor, trained = case["rotary"], case["scaling"], case["factor"], case["original"]
    f = np.empty(d // 2)
    turn = 2 * math.pi

    def index_of(turns):  # the place whose wave turns so often over the trained length
        return d * math.log(trained / (turns * turn)) / (2 * math.log(BASE))

    for i in range(d // 2):
        f[i] = math.exp(-2 * i / d * math.log(BASE))
        if kind == "linear":
            f[i] /= factor
        elif kind == "ntk":
            f[i] *= factor ** (-2 * i / (d - 2))
        elif kind == "ramp":
            a, b = max(math.floor(index_of(32)), 0), min(math.ceil(index_of(1)), d - 1)
            p = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f[i] *= p / factor + 1 - p
        elif kind == "bands":
            p = min(max((trained / (turn / f[i]) - 1) / (4 - 1), 0.0), 1.0)
            f[i] *= (1 - p) / factor + p
    a = (int(seed) % 1000 + np.arange(case["rows"], dtype=np.float64))[:, None] * f
    return {"cos": torch.from_numpy(np.cos(a)), "sin": torch.from_numpy(np.sin(a))}


def _turn(layout, x, c, s, r):
    """A complex product: element pairs of the first r times c + i s."""
    one, two = ((slice(0, r, 2), slice(1, r, 2)) if layout == "pairs"
                else (slice(0, r // 2), slice(r // 2, r)))
    z = (x[..., one] + 1j * x[..., two]) * (c.astype(np.float64) + 1j * s.astype(np.float64))
    y = x.copy()
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_rows(case, s, b, x, rotary):
    """The first counts[b] rows of x [heads, tokens, dim], rotated."""
    n, at = s["counts"][b], int(s["starts"][b])
    return _turn(case["layout"], x[:, :n], s["cos"].cpu().numpy()[at:at + n],
                 s["sin"].cpu().numpy()[at:at + n], rotary)


def _held(case, x, scale):
    """Numbers as a page's type can hold them, before they are rounded to it."""
    return np.clip(x / np.float64(np.float32(scale)), -448, 448) if case["dtype"] == "fp8" else x


def _numbers(case, pool):
    if case["dtype"] == "fp8":
        pool = pool.view(torch.float8_e4m3fn)
    return pool.to(torch.float32).cpu().numpy().astype(np.float64)


def _host(x):
    return x.cpu().numpy().astype(np.float64)


def _exact_append(case, s):
    q, k, v = _host(s["q"]), _host(s["k"]), _host(s["v"])
    kp, vp = _numbers(case, s["kp"]), _numbers(case, s["vp"])
    out = [np.zeros(x.shape) for x in (q, k, v)]
    slots = s["slots"].cpu().numpy()
    for b, n in enumerate(s["counts"]):
        out[0][b, :, :n] = _exact_rows(case, s, b, q[b], case["rotary"])
        out[1][b, :, :n] = _exact_rows(case, s, b, k[b], case["rotary"])
        out[2][b, :, :n] = v[b, :, :n]
        for t in range(n):
            page, row = divmod(int(slots[b, t]), P)
            kp[page, :, row] = _held(case, out[1][b, :, t], K_SCALE)
            vp[page, :, row] = _held(case, v[b, :, t], V_SCALE)
    q, k, v, kp, vp = (torch.from_numpy(x) for x in (*out, kp, vp))
    return {"q": q, "k": k, "v": v, "keys": kp, "values": vp}


def _exact_latent_append(case, s):
    q, latent, rope_key = _host(s["q"]), _host(s["latent"]), _host(s["rope_key"])
    pool, out = _numbers(case, s["pool"]), np.zeros(q.shape)
    slots = s["slots"].cpu().numpy()
    for b, n in enumerate(s["counts"]):
        out[b, :, :n] = _exact_rows(case, s, b, q[b], ROPE)
        turned = _exact_rows(case, s, b, rope_key[b][None], ROPE)[0]
        for t in range(n):
            page, row = divmod(int(slots[b, t]), P)
            pool[page, row] = _held(case, np.concatenate([latent[b, t], turned[t]]), K_SCALE)
    return {"q": torch.from_numpy(out), "pages": torch.from_numpy(pool)}


def _exact_latent(case, s):
    """A sequence after another: softmax over the tokens that a row sees."""
    n, hq, t = case["latent"], case["q_heads"], case["tokens"]
    out = torch.zeros(case["batch"], hq, t, n, dtype=torch.float64, device=DEV)
    for b, (length, count) in enumerate(zip(s["host_lengths"], s["counts"])):
        x = s["pool"].index_select(0, s["tables"][b][:-(-length // P)].long())
        if case["dtype"] == "fp8":  # the scale is an fp32 number, the product a 64-bit one
            x = x.view(torch.float8_e4m3fn).double() * float(np.float32(K_SCALE))
        rows = x.double().flatten(0, 1)
        for i in range(count):
            seen = rows[:length - count + i + 1]
            w = torch.softmax(s["q"][b, :, i].double() @ seen.T * _softmax_scale(case), dim=1)
            out[b, :, i] = w @ seen[:, :n]
    return out


def _exact_expanded(case, s):
    """A head of a sequence after another."""
    h, t = case["heads"], case["tokens"]
    out = torch.zeros(case["batch"], h, t, NOPE, dtype=torch.float64, device=DEV)
    for b, (end, count) in enumerate(zip(s["key_counts"], s["counts"])):
        if count == 0:
            continue
        later = torch.ones(count, end, dtype=torch.bool, device=DEV).triu(end - count + 1)
        shared = s["rope_key"][b, :end].double()
        for i in range(h):
            q = s["q"][b, i, :count].double()
            x = q[:, :NOPE] @ s["k"][b, i, :end].double().T + q[:, NOPE:] @ shared.T
            w = torch.softmax((x * _softmax_scale(case)).masked_fill(later, -math.inf), dim=1)
            out[b, i, :count] = w @ s["v"][b, i, :end].double()
    return out
