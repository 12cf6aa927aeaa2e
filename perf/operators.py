"""Performance cases of tree decoding over the paged cache: the step of a
server that lets a target model check a tree of drafted tokens at once.

A case's "kind" says which operator it stands for:

- "attention": one layer's attention of such a step (paged_tree_attention).
  Each sequence has a paged history and a tree of nodes; node 0 holds the last
  token that was generated, the others drafted tokens.  A node's query sees the
  whole history, its ancestors in the tree and itself.
- "verify": which drafted tokens the target's probabilities let pass, by given
  random numbers, and the token that follows them (verify_tree).
- "append": the K/V rows of the nodes that passed, taken out of the tree's
  rows of all layers and written to their places in the pages (append_path).

With `own` false the operators run in their plain forms, with it true through
the framework's entry points.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
D, P = 128, 16  # head size and page size of the batched entry points
K_SCALE, V_SCALE = 0.03, 0.015  # fp8 scales of a calibrated cache (448 * scale covers the rows)


# ------------------------------------------------------------------ cases ----
def listed():
    return [
        # One chat at its beginning with a small tree: launches and latency.
        dict(name="attend_small", kind="attention", batch=1, q_heads=32, kv_heads=8, nodes=5,
             low=121, high=121, ragged=False, chain=False, dtype="bf16"),
        # One chat over a very long context.
        dict(name="attend_long", kind="attention", batch=1, q_heads=32, kv_heads=8, nodes=33,
             low=131071, high=131071, ragged=False, chain=False, dtype="bf16"),
        # No head grouping (32/32 heads), a chain of drafts per sequence.
        dict(name="attend_mha", kind="attention", batch=8, q_heads=32, kv_heads=32, nodes=7,
             low=128, high=2048, ragged=False, chain=True, dtype="f32"),
        # A full server: 64 sequences, contexts log-uniform in [512, 8192], on
        # fp32 and bf16 pages; the trees of the second have their own sizes.
        dict(name="attend_f32", kind="attention", batch=64, q_heads=32, kv_heads=8, nodes=16,
             low=512, high=8192, ragged=False, chain=False, dtype="f32"),
        dict(name="attend_bf16", kind="attention", batch=64, q_heads=32, kv_heads=8, nodes=16,
             low=512, high=8192, ragged=True, chain=False, dtype="bf16"),
        # The widest trees, on fp8 pages: the most arithmetic.
        dict(name="attend_wide", kind="attention", batch=64, q_heads=32, kv_heads=8, nodes=64,
             low=512, high=8192, ragged=False, chain=False, dtype="fp8"),
        # One chat with a chain of sampled drafts.
        dict(name="verify_chain", kind="verify", batch=1, nodes=6, vocab=32000, rows=True,
             ragged=False, chain=True),
        # 64 sequences with trees of a drafter's most likely tokens.
        dict(name="verify_likely", kind="verify", batch=64, nodes=16, vocab=128256, rows=False,
             ragged=False, chain=False),
        # 64 sequences with trees of sampled drafts, whose distributions count.
        dict(name="verify_sampled", kind="verify", batch=64, nodes=16, vocab=128256, rows=True,
             ragged=True, chain=False),
        # One chat's accepted tokens, 32 layers of bf16 pages.
        dict(name="append_one", kind="append", layers=32, batch=1, kv_heads=8, nodes=5,
             ragged=False, dtype="bf16"),
        # A full server's accepted tokens in 32 layers of fp32 and bf16 pages.
        dict(name="append_f32", kind="append", layers=32, batch=64, kv_heads=8, nodes=16,
             ragged=False, dtype="f32"),
        dict(name="append_bf16", kind="append", layers=32, batch=64, kv_heads=8, nodes=33,
             ragged=True, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "verify", "verify", "append"])
    nodes = rng.choice([_log_int(rng, 1, 64), _log_int(rng, 2, 32)])
    ragged = rng.random() < 0.4
    if kind == "attention":
        kv_heads, group = rng.choice([(8, 4), (8, 4), (8, 1), (32, 1), (4, 8), (16, 2), (8, 5),
                                      (2, 16)])
        batch = _log_int(rng, 1, 64)
        high = _log_int(rng, 16, 8192 if kv_heads <= 8 else 2048)
        if batch == 1 and rng.random() < 0.5:
            high = _log_int(rng, 8192, 131071)
        low = rng.choice([high, high // 4, high // 16, 0])
        return dict(kind="attention", batch=batch, q_heads=kv_heads * group, kv_heads=kv_heads,
                    nodes=nodes, low=low, high=high, ragged=ragged, chain=rng.random() < 0.3,
                    dtype=rng.choice(["f32", "bf16", "fp8"]))
    if kind == "verify":
        batch = _log_int(rng, 1, 64)
        vocab = _log_int(rng, 100, 128256)
        return dict(kind="verify", batch=batch, nodes=min(nodes, 1024 // batch), vocab=vocab,
                    rows=rng.random() < 0.6, ragged=ragged, chain=rng.random() < 0.4)
    return dict(kind="append", layers=_log_int(rng, 1, 32), batch=_log_int(rng, 1, 64),
                kv_heads=rng.choice([1, 3, 8, 8]), nodes=min(nodes, 33), ragged=ragged,
                dtype=rng.choice(["f32", "bf16"]))


# ----------------------------------------------------------------- inputs ----
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _rand(g, *shape):
    return torch.rand(*shape, device=DEV, generator=g)


def _case_rng(case, salt):
    return np.random.default_rng([salt, case["batch"], case["nodes"], case.get("high", 0),
                                  case.get("vocab", 0), case.get("layers", 0)])


def _lengths(case):
    """The batch's context lengths: part of the case, the same for every seed."""
    low, high, n = case["low"], case["high"], case["batch"]
    rng = _case_rng(case, 1)
    if low > 0 and high > 4 * low:  # contexts of a batch spread over their logarithm
        v = np.exp(rng.uniform(math.log(low), math.log(high + 1), size=n)).astype(np.int64)
        return [int(min(high, max(low, x))) for x in v]
    return [int(x) for x in rng.integers(min(low, high), high + 1, size=n)]


def _counts(case):
    """Nodes of each sequence's tree (part of the case)."""
    b, t = case["batch"], case["nodes"]
    if not case["ragged"]:
        return [t] * b
    return [int(x) for x in _case_rng(case, 2).integers(min(1, t // 2), t + 1, size=b)]


def _accepted(case):
    """Accepted nodes of each sequence of an append case (part of the case):
    mostly a few, as drafts pass."""
    counts = _counts(case)
    v = 1 + _case_rng(case, 3).geometric(0.3, size=len(counts))
    return [int(min(x, c)) for x, c in zip(v, counts)]


def _parents(case, seed):
    """[batch, nodes] parents, -1 for the root: chains, or trees whose nodes
    hang from one of the nodes shortly before them."""
    b, t = case["batch"], case["nodes"]
    out = np.arange(-1, t - 1, dtype=np.int32)[None].repeat(b, 0)
    if not case["chain"]:
        rng = np.random.default_rng(int(seed) + 77)
        for i in range(1, t):
            out[:, i] = rng.integers(max(0, (i - 1) // 3), min(i, max(1, (i + 1) // 2 + 1)), size=b)
    return out


def _i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=DEV)


def _on_pages(dtype, x, scale):
    """fp32 rows as their pages hold them, in fp32."""
    if dtype == "bf16":
        return x.to(torch.bfloat16).to(torch.float32)
    if dtype == "fp8":
        by = torch.full((), scale, device=x.device)  # a tensor: a true fp32 division
        codes = (x / by).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return codes.to(torch.float32) * by
    return x


def _pool(g, dtype, scale, channel, *shape):
    """Pages [N, Hkv, 16, 128] of random rows in their element type."""
    x = _randn(g, *shape)
    if channel is not None:
        x *= channel
    if dtype == "bf16":
        return x.to(torch.bfloat16)
    if dtype == "fp8":
        return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return x


def _attention_inputs(case, seed):
    g = _generator(seed)
    b, hq, hkv, t = case["batch"], case["q_heads"], case["kv_heads"], case["nodes"]
    lengths = _lengths(case)
    pages = [(n + P - 1) // P for n in lengths]
    physical = sum(pages) + 3
    channel = torch.exp(0.4 * _randn(g, hkv, 1, D))  # keys differ in size by channel
    kp = _pool(g, case["dtype"], K_SCALE, channel, physical, hkv, P, D)
    vp = _pool(g, case["dtype"], V_SCALE, None, physical, hkv, P, D)
    order = np.random.default_rng(int(seed) + 5).permutation(physical)
    tables = np.zeros((b, max(1, max(pages))), np.int32)
    at = 0
    for i, n in enumerate(pages):
        tables[i, :n] = order[at:at + n]
        at += n
    return dict(q=_randn(g, b, hq, t, D), kp=kp, vp=vp, tables=_i32(tables),
                lengths=_i32(lengths), tk=(_randn(g, b, hkv, t, D) * channel).contiguous(),
                tv=_randn(g, b, hkv, t, D), parents=_parents(case, seed), counts=_counts(case),
                host_lengths=lengths)


def _verify_inputs(case, seed):
    """Probabilities of the target and of a drafter that knows it fairly well,
    and the drafter's tokens: drawn from its rows, or its most likely ones."""
    g = _generator(seed)
    b, t, v = case["batch"], case["nodes"], case["vocab"]
    logits = _randn(g, b, t, v) * 2.5
    logits[..., :: max(1, v // 8)] += 6.0  # a few tokens carry much of the mass
    target = torch.softmax(logits, dim=-1)
    logits += 0.6 * _randn(g, b, t, v)
    draft = torch.softmax(logits, dim=-1)
    parents = _parents(case, seed)
    at = torch.as_tensor(np.maximum(parents, 0), device=DEV).long()
    if case["rows"]:
        # One draw per node from its parent's row, by exponential races.
        tokens = torch.empty(b, t, dtype=torch.int32, device=DEV)
        for c in range(t):
            q = draft[torch.arange(b, device=DEV), at[:, c]]
            race = -torch.log(_rand(g, b, v).clamp_min(1e-30))
            tokens[:, c] = torch.argmax(q / race, dim=-1).to(torch.int32)
    else:
        rank = np.zeros((b, t), np.int64)  # which child of its parent a node is
        for i in range(1, t):
            rank[:, i] = (parents[:, 1:i] == parents[:, i:i + 1]).sum(1)
        k = min(v, int(rank.max()) + 1)
        best = torch.topk(draft, k, dim=-1).indices
        r = torch.as_tensor(np.minimum(rank, k - 1), device=DEV)
        tokens = best[torch.arange(b, device=DEV)[:, None], at, r].to(torch.int32)
        draft = None
    return dict(target=target, draft=draft, tokens=tokens.contiguous(), parents=parents,
                uniforms=_rand(g, b, t), bonus=_rand(g, b), counts=_counts(case))


def _append_inputs(case, seed):
    g = _generator(seed)
    n_layers, b, hkv, t = case["layers"], case["batch"], case["kv_heads"], case["nodes"]
    each = (t + 2 * P - 2) // P  # pages a sequence's reserved slots can touch
    physical = b * each + 2
    kp = _pool(g, case["dtype"], 1.0, None, n_layers, physical, hkv, P, D)
    vp = _pool(g, case["dtype"], 1.0, None, n_layers, physical, hkv, P, D)
    rng = np.random.default_rng(int(seed) + 6)
    order = rng.permutation(physical)
    slots = np.zeros((b, t), np.int64)
    path = np.full((b, t), -1, np.int32)
    accepted = _accepted(case)
    counts = _counts(case)
    for i in range(b):
        pos = int(rng.integers(0, P)) + np.arange(t)
        slots[i] = order[i * each + pos // P].astype(np.int64) * P + pos % P
        if accepted[i]:
            later = np.sort(rng.choice(np.arange(1, max(2, counts[i])), accepted[i] - 1,
                                       replace=False))
            path[i, :accepted[i]] = np.concatenate([[0], later])
    return dict(k=_randn(g, n_layers, b, hkv, t, D), v=_randn(g, n_layers, b, hkv, t, D), kp=kp,
                vp=vp, slots=torch.as_tensor(slots, device=DEV), path=_i32(path),
                accepted=_i32(accepted))


def _inputs(case, seed):
    return {"attention": _attention_inputs, "verify": _verify_inputs,
            "append": _append_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s.update(kind=case["kind"], dtype=case.get("dtype"))
    if "parents" in s:
        s["host_parents"] = s["parents"]
        s["parents"] = _i32(s["parents"])
        s["node_counts"] = _i32(s["counts"]) if case["ragged"] else None
    b, t = case["batch"], case["nodes"]
    if case["kind"] == "attention":
        s["out"] = torch.zeros_like(s["q"])  # rows behind a tree's last node stay 0
        if own:
            import helix_runtime_amd as hx
            s["workspace"] = hx.tree_workspace(b, case["q_heads"], case["kv_heads"], t)
        else:
            # [batch, nodes, nodes]: whether a node sees another, as a server
            # keeps it beside the parents.
            s["seen"] = torch.as_tensor(_ancestors(s["host_parents"]), device=DEV)
            s["live"] = (torch.arange(t, device=DEV)[None] < _i32(s["counts"])[:, None])
    elif case["kind"] == "verify":
        s["path"] = torch.empty(b, t, dtype=torch.int32, device=DEV)
        s["accepted"] = torch.empty(b, dtype=torch.int32, device=DEV)
        s["next"] = torch.empty(b, dtype=torch.int32, device=DEV)
        if own:
            import helix_runtime_amd as hx
            s["workspace"] = hx.verify_workspace(b, t, case["vocab"])
    return s


def _ancestors(parents):
    b, t = parents.shape
    seen = np.zeros((b, t, t), bool)
    rows = np.arange(b)
    for i in range(t):
        up = parents[:, i]
        seen[:, i] = np.where((up >= 0)[:, None], seen[rows, np.maximum(up, 0)], False)
        seen[:, i, i] = True
    return seen


# -------------------------------------------------------------------- run ----
def run(s):
    if s["kind"] == "attention":
        return _run_attention_own(s) if own else _run_attention(s)
    if s["kind"] == "verify":
        return _run_verify_own(s) if own else _run_verify(s)
    return _run_append_own(s) if own else _run_append(s)


def _run_attention_own(s):
    import helix_runtime_amd as hx
    hx.paged_tree_attention(s["q"], s["kp"], s["vp"], s["tables"], s["lengths"], s["tk"], s["tv"],
                            s["parents"], s["out"], s["workspace"], node_counts=s["node_counts"],
                            page_dtype=s["dtype"], k_scale=K_SCALE, v_scale=V_SCALE)
    return s["out"]


def _widened(s, pool, scale):
    if s["dtype"] == "fp8":
        return pool.view(torch.float8_e4m3fn).to(torch.float32) * scale
    return pool.to(torch.float32)


def _run_attention(s):
    q, out = s["q"], s["out"]
    _, hq, t, d = q.shape
    hkv = s["tk"].shape[1]
    group = hq // hkv
    tk = _on_pages(s["dtype"], s["tk"], K_SCALE)
    tv = _on_pages(s["dtype"], s["tv"], V_SCALE)
    for b, n in enumerate(s["host_lengths"]):
        pages = s["tables"][b, :(n + P - 1) // P].long()
        k = _widened(s, s["kp"][pages], K_SCALE).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        v = _widened(s, s["vp"][pages], V_SCALE).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        k, v = torch.cat([k, tk[b]], dim=1), torch.cat([v, tv[b]], dim=1)
        x = torch.matmul(q[b].reshape(hkv, group * t, d), k.transpose(1, 2).contiguous())
        x = x.view(hkv, group, t, n + t) / math.sqrt(d)
        x[..., n:].masked_fill_(~s["seen"][b], -math.inf)
        x = torch.exp(x - x.amax(dim=-1, keepdim=True))
        y = torch.matmul(x.view(hkv, group * t, n + t), v).view(hkv, group, t, d)
        y = (y / x.sum(dim=-1, keepdim=True)).reshape(hq, t, d)
        out[b] = torch.where(s["live"][b][None, :, None], y, out[b])
    return out


def _run_verify_own(s):
    import helix_runtime_amd as hx
    hx.verify_tree(s["target"], s["draft"], s["tokens"], s["parents"], s["uniforms"], s["bonus"],
                   s["path"], s["accepted"], s["next"], s["workspace"],
                   node_counts=s["node_counts"])
    return {"path": s["path"], "accepted": s["accepted"], "next": s["next"]}


def _run_verify(s):
    """All sequences side by side, the nodes in order: a node whose parent is
    the last accepted one is tried, and either accepted or taken out of the
    row that is left.  In 64 bits: what is accepted hangs on comparisons."""
    target, draft, tokens, parents = s["target"], s["draft"], s["tokens"], s["parents"]
    b, t, v = target.shape
    counts = s["node_counts"]
    if counts is None:
        counts = torch.full((b,), t, dtype=torch.int32, device=DEV)
    each = torch.arange(b, device=DEV)
    cur = torch.zeros(b, dtype=torch.long, device=DEV)
    number = (counts > 0).long()
    path = torch.full((b, t + 1), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = torch.where(counts > 0, 0, -1)
    left = target[:, 0].double()
    mass = torch.ones(b, dtype=torch.float64, device=DEV)
    for c in range(1, t):
        tried = (parents[:, c] == cur) & (counts > c) & (tokens[:, c] >= 0) & (tokens[:, c] < v)
        x = tokens[:, c].long().clamp(0, v - 1)
        have = left[each, x]
        u = s["uniforms"][:, c].double()
        if draft is not None:
            q = draft[each, cur].double()
            passed = tried & (u * q[each, x] < have)
            rest = (left - q).clamp_min(0.0)
            total = rest.sum(dim=-1)
            rest = rest / torch.where(total > 0, total, 1.0)[:, None]
        else:
            passed = tried & (u * mass < have)
            rest = left.clone()
            rest[each, x] = 0.0
            mass = torch.where(tried & ~passed, mass - have, mass)
        failed = tried & ~passed
        left = torch.where(passed[:, None], target[:, c].double(),
                           torch.where(failed[:, None], rest, left))
        mass = torch.where(passed, 1.0, mass)
        path[each, torch.where(passed, number, t)] = c
        number = number + passed
        cur = torch.where(passed, c, cur)
    left = torch.where((left.sum(dim=-1) > 0)[:, None], left, target[each, cur].double())
    sums = left.cumsum(dim=-1)
    after = (sums <= s["bonus"].double()[:, None] * sums[:, -1:]).sum(dim=-1)
    last = (torch.arange(v, device=DEV) * (left > 0)).amax(dim=-1)  # where rounding goes past it
    after = torch.where(counts > 0, torch.minimum(after, last), -1)
    return {"path": path[:, :t].contiguous(), "accepted": number.to(torch.int32),
            "next": after.to(torch.int32)}


def _run_append_own(s):
    import helix_runtime_amd as hx
    hx.append_path(s["k"], s["v"], s["kp"], s["vp"], s["slots"], s["path"], s["accepted"],
                   page_dtype=s["dtype"])
    return {"keys": s["kp"], "values": s["vp"]}


def _run_append(s):
    b, t = s["slots"].shape
    page, row = s["slots"] // P, s["slots"] % P
    taken = (torch.arange(t, device=DEV)[None] < s["accepted"][:, None])[:, :, None, None, None]
    node = s["path"].long().clamp_min(0)
    each = torch.arange(b, device=DEV)[:, None]
    for src, pool in ((s["k"], s["kp"]), (s["v"], s["vp"])):
        rows = src[:, each, :, node].to(pool.dtype)  # [batch, nodes, layers, heads, dim]
        pool[:, page, :, row] = torch.where(taken, rows, pool[:, page, :, row])
    return {"keys": s["kp"], "values": s["vp"]}


# ------------------------------------------------------------------- work ----
def work(case):
    b, t = case["batch"], case["nodes"]
    if case["kind"] == "verify":
        # The tried entries, and the row that the following token is drawn from.
        row = case["vocab"] * 4 * (2 if case["rows"] else 1)
        return {"bytes": b * (row + 8 * t + 12 * t + 12), "flops": 4 * b * case["vocab"]}
    size = {"f32": 4, "bf16": 2, "fp8": 1}[case["dtype"]]
    hkv = case["kv_heads"]
    if case["kind"] == "append":
        rows = 2 * case["layers"] * hkv * D * sum(_accepted(case))
        return {"bytes": rows * (4 + size) + 12 * b * t, "flops": 0}
    hq = case["q_heads"]
    lengths, counts = _lengths(case), _counts(case)
    nodes = sum(counts)
    pairs = sum(c * (n + (c + 1) / 2) for n, c in zip(lengths, counts))
    return {"bytes": 2 * hkv * D * (size * sum(lengths) + 4 * nodes) + 8 * hq * D * nodes,
            "flops": int(4 * hq * D * pairs)}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    if case["kind"] == "verify":
        return _exact_verify(case, s)
    for src, name in ((s["k"], "kp"), (s["v"], "vp")):
        pool = s[name].double()
        flat = pool.transpose(2, 3).contiguous().view(pool.shape[0], -1, pool.shape[2], D)
        path = s["path"].tolist()
        for b, n in enumerate(s["accepted"].tolist()):
            for i in range(n):
                row = src[:, b, :, path[b][i]]
                flat[:, int(s["slots"][b, i])] = _on_pages(case["dtype"], row, 1.0).double()
        s[name] = flat.view(pool.shape[0], pool.shape[1], P, pool.shape[2], D).transpose(2, 3)
    return {"keys": s["kp"].contiguous(), "values": s["vp"].contiguous()}


def _exact_attention(case, s):
    """Row by row of the definition: softmax over the keys that a node sees."""
    hq, hkv, t = case["q_heads"], case["kv_heads"], case["nodes"]
    dtype = case["dtype"]
    out = torch.zeros(case["batch"], hq, t, D, dtype=torch.float64, device=DEV)

    def pages(pool, ids, scale):
        x = pool.index_select(0, ids)
        if dtype == "fp8":
            # The scale is an fp32 number, the product a 64-bit one.
            x = x.view(torch.float8_e4m3fn).double() * float(np.float32(scale))
        return x.double().permute(1, 0, 2, 3).flatten(1, 2)

    for b, (n, count) in enumerate(zip(s["host_lengths"], s["counts"])):
        ids = s["tables"][b][:-(-n // P)].long()
        k, v = pages(s["kp"], ids, K_SCALE)[:, :n], pages(s["vp"], ids, V_SCALE)[:, :n]
        kt = _on_pages(dtype, s["tk"][b], K_SCALE).double()
        vt = _on_pages(dtype, s["tv"][b], V_SCALE).double()
        hidden = torch.zeros(t, t, dtype=torch.float64, device=DEV)
        for i in range(t):
            line, at = set(), i
            while at >= 0:
                line.add(at)
                at = int(s["parents"][b][at])
            hide = [j for j in range(t) if j not in line]
            if hide:
                hidden[i, hide] = -math.inf
        for h in range(hq):
            q = s["q"][b, h].double() * D ** -0.5
            kk, vv = h // (hq // hkv), h // (hq // hkv)
            x = torch.cat([q @ k[kk].T, q @ kt[kk].T + hidden], dim=1)
            w = torch.softmax(x, dim=1)
            out[b, h] = w[:, :n] @ v[vv] + w[:, n:] @ vt[vv]
        out[b, :, count:] = 0
    return out


def _exact_verify(case, s):
    """Sequence by sequence: a walk from the root."""
    b, t, v = case["batch"], case["nodes"], case["vocab"]
    path = np.full((b, t), -1, np.int32)
    accepted, after = np.zeros(b, np.int32), np.full(b, -1, np.int32)
    tokens, u = s["tokens"].cpu().numpy(), s["uniforms"].double().cpu().numpy()
    bonus = s["bonus"].double().cpu().numpy()

    def host(x):
        return x.cpu().numpy().astype(np.float64)

    for i in range(b):
        if s["counts"][i] == 0:
            continue
        at, way = 0, [0]
        while True:
            left, mass = host(s["target"][i, at]), 1.0
            q = host(s["draft"][i, at]) if s["draft"] is not None else None
            went = None
            for c in range(at + 1, s["counts"][i]):
                x = int(tokens[i, c])
                if s["parents"][i, c] != at or not 0 <= x < v:
                    continue
                if u[i, c] * (mass if q is None else q[x]) < left[x]:
                    went = c
                    break
                if q is None:
                    mass -= left[x]
                    left[x] = 0.0
                else:
                    left = np.maximum(left - q, 0.0)
                    total = math.fsum(left)
                    left = left / total if total > 0 else left
            if went is None:
                break
            at = went
            way.append(at)
        if not left.sum() > 0:
            left = host(s["target"][i, at])
        sums = np.cumsum(left)
        k = int(np.searchsorted(sums, bonus[i] * sums[-1], side="right"))
        after[i] = min(k, int(np.flatnonzero(left > 0)[-1]))
        accepted[i] = len(way)
        path[i, :len(way)] = way
    return {"path": torch.from_numpy(path), "accepted": torch.from_numpy(accepted),
            "next": torch.from_numpy(after)}
