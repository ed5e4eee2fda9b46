"""Cases that measure the cache and low-bit operators of the library: attention
of a tree of drafted tokens over a KV cache, the attention weight that each
cached token has collected, commit of an accepted path into the cache, eviction
by collected weight, and products with 4-bit weights.

`own = False` computes every operator in its plain form (torch operations);
`own = True` calls mrtops, the ctypes bindings of libmrtdf.so.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "magenta-realtime-mlx-cpp_b200")
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
# No case reads, writes or computes more than the largest listed ones.
MOST_BYTES, MOST_FLOPS, MOST_SCORES = 5.6e8, 3.5e10, 1.6e8


def _ops():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import mrtops

    return mrtops


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # One CFG pair verifies a tree of 16 drafted frames against the temporal
        # self-attention cache (50 frames, T5 position bias): latency.
        dict(name="tree self 2x16 n16", op="tree", dtype="bf16", B=2, H=16, KV=16, D=64, N=16, cap=50, low=20, high=50,
             bias=128, evicted=False, packed=True, pad=0.0),
        # One token per row over a context of 1006 for 64 CFG pairs: the wide
        # streams' decode step, bound by the cache.
        dict(name="token 128x16 ctx1006", op="tree", dtype="bf16", B=128, H=16, KV=16, D=64, N=1, cap=1006, low=1006,
             high=1006, bias=0, evicted=False, packed=False, pad=0.0),
        # float32 engine, a small tree over an evicted cache (positions stored).
        dict(name="tree fp32 2x16 n8", op="tree", dtype="fp32", B=2, H=16, KV=16, D=64, N=8, cap=1006, low=700,
             high=1006, bias=128, evicted=True, packed=False, pad=0.0),
        # Grouped heads, long ragged caches, an odd tree with padded nodes.
        dict(name="tree gqa 4x32/8 n24 16k", op="tree", dtype="bf16", B=4, H=32, KV=8, D=128, N=24, cap=16384,
             low=4097, high=16360, bias=0, evicted=False, packed=True, pad=0.2),
        # Weight collected after a short verification, float32.
        dict(name="mass fp32 2x16", op="mass", dtype="fp32", L=1, B=2, H=16, KV=16, D=64, N=8, cap=256, low=90, high=250,
             bias=128, evicted=True, path=3),
        # The same over long grouped caches of two layers.
        dict(name="mass gqa 2x8x32/8 8k", op="mass", dtype="bf16", L=2, B=8, H=32, KV=8, D=128, N=16, cap=8192, low=3001,
             high=8190, bias=0, evicted=False, path=5),
        # An accepted path of all 20 temporal layers of one CFG pair.
        dict(name="commit 20x2x16", op="commit", dtype="bf16", L=20, B=2, KV=16, D=64, N=16, cap=50, low=8, high=44,
             path=5, evicted=True),
        # The same for 32 rows of a wide float32 stream.
        dict(name="commit fp32 32x32x8", op="commit", dtype="fp32", L=32, B=32, KV=8, D=128, N=64, cap=256, low=100,
             high=240, path=12, evicted=True),
        # One frame over budget in the temporal cache.
        dict(name="evict 2x16 50->40", op="evict", dtype="bf16", L=1, B=2, KV=16, D=64, cap=50, low=41, high=50,
             budget=40, recent=8, sinks=1),
        # Compaction of long prompts to an eighth.
        dict(name="evict 4x4x8 16k->2k", op="evict", dtype="bf16", L=4, B=4, KV=8, D=128, cap=16384, low=9000, high=16384,
             budget=2048, recent=256, sinks=4),
        # The vocabulary projection of one CFG pair, float32 activations.
        dict(name="q4 fp32 2x16388x1024", op="q4", dtype="fp32", M=2, N=16388, K=1024, group=64, out="fp32"),
        # A wide projection of eight rows.
        dict(name="q4 bf16 8x16384x8192", op="q4", dtype="bf16", M=8, N=16384, K=8192, group=128, out="bf16"),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "mass", "commit", "evict", "q4"])
    while True:
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp32"]))
        if op == "q4":
            c.update(M=_log(rng, 1, 64), group=rng.choice([32, 64, 128]), N=_log(rng, 64, 32768))
            c.update(K=c["group"] * _log(rng, 2, 12288 // c["group"]), out=rng.choice([c["dtype"], "fp32"]))
        else:
            kv, g = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4, 8])
            cap = _log(rng, 24, 32768)
            c.update(B=_log(rng, 1, 64), KV=kv, D=rng.choice([64, 128]), cap=cap)
            high = rng.randint(max(1, cap // 2), cap)
            low = rng.choice([0, high, high // 2, high // 8])
            if op == "evict":
                budget = _log(rng, 8, cap)
                recent = rng.randint(0, budget // 2)
                c.update(L=_log(rng, 1, 16), low=low, high=high, budget=budget, recent=recent,
                         sinks=rng.randint(0, min(8, budget - recent)))
            else:
                c.update(N=_log(rng, 1, 64), evicted=rng.choice([True, False]))
                if op == "commit":
                    c.update(L=_log(rng, 1, 32), path=rng.randint(1, c["N"]), low=min(low, max(0, cap - c["N"])),
                             high=max(0, min(high, cap - c["N"])))
                else:
                    c.update(H=kv * g, low=low, high=high, bias=rng.choice([0, 16, 128]))
                    if op == "mass":
                        c.update(L=_log(rng, 1, 4), path=rng.randint(1, min(16, c["N"])), high=max(0, min(high, cap - c["N"])))
                        c["low"] = min(low, c["high"])
                    else:
                        c.update(packed=rng.choice([True, False]), pad=rng.choice([0.0, 0.2]))
        w = work(c)
        scores = c["B"] * c.get("H", 0) * c.get("N", 0) * c["cap"] * c.get("L", 1) if op in ("tree", "mass") else 0
        held = c.get("L", 1) * c["B"] * c["KV"] * c["cap"] * c["D"] * 2 * BYTES[c["dtype"]] if op != "q4" else 0
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and scores <= MOST_SCORES and held <= 2e9 and w["bytes"] >= 1e4:
            return c


def _lens(c):
    """Expected rows in use over all sequences: a uniform draw of low .. high."""
    return c["B"] * (c["low"] + c["high"]) / 2


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "q4":
        m, n, k = c["M"], c["N"], c["K"]
        return {"bytes": n * k / 2 + 2 * e * n * k / c["group"] + m * k * e + m * n * BYTES[c["out"]], "flops": 2.0 * m * n * k}
    d, kv, t = c["D"], c["KV"], _lens(c)
    if c["op"] == "tree":
        n, b, h = c["N"], c["B"], c["H"]
        read = kv * d * e * 2 * (t + b * n) + (4 * kv * t if c["evicted"] and c["bias"] else 0)
        return {"bytes": read + 2 * b * h * n * d * e + 4 * b * h * n, "flops": 4.0 * h * n * d * (t + b * n / 2)}
    if c["op"] == "mass":
        p, b, h = c["path"], c["B"], c["H"]
        read = kv * d * e * (t + b * p) + (4 * kv * t if c["evicted"] and c["bias"] else 0) + b * h * p * (d * e + 4)
        return {"bytes": c["L"] * (read + 4 * kv * (2 * t + b * p)), "flops": 2.0 * c["L"] * h * p * d * (t + b * p)}
    if c["op"] == "commit":
        rows = c["L"] * c["B"] * kv * c["path"] * 0.5
        return {"bytes": rows * (4 * d * e + 4), "flops": rows * d}
    over = max(0.0, 1 - c["budget"] / max(1.0, c["high"]))
    kept = c["L"] * kv * c["B"] * c["budget"]
    return {"bytes": 8 * c["L"] * kv * t + 8 * kept + kept * over * 4 * d * e, "flops": 8.0 * c["L"] * kv * t}


# ---- inputs --------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _uniform_int(g, low, high, *shape):
    """Whole numbers low .. high, both included."""
    return (low + (torch.rand(*shape, generator=g, device="cuda") * (high - low + 1)).floor().clamp_(max=high - low)).to(torch.int32)


def _evicted_positions(g, shape, lens, gap=8):
    """Positions of what an evicted cache still holds: distinct, not in slot order
    everywhere, below next_pos = gap * capacity."""
    cap = shape[-1]
    pos = torch.arange(cap, device="cuda", dtype=torch.int32) * gap + _uniform_int(g, 0, gap - 1, *shape)
    half = cap // 2
    pos[..., :half] = pos[..., :half].flip(-1)
    return pos, torch.full_like(lens, gap * cap)


def prepare(c, seed):
    g, t = _gen(seed), TYPES[c["dtype"]]
    s = dict(c=c)
    if c["op"] == "q4":
        m, n, k, gr = c["M"], c["N"], c["K"], c["group"]
        s["x"] = _normal(g, m, k, dtype=t)
        s["packed"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (torch.rand(n, k // gr, generator=g, device="cuda") * 0.004 + 0.004).to(t)
        s["biases"] = (s["scales"].float() * -(7.5 + _normal(g, n, k // gr, std=0.5))).to(t)
        return s
    b, kv, d, cap = c["B"], c["KV"], c["D"], c["cap"]
    s["lens"] = _uniform_int(g, c["low"], c["high"], b)
    lead = (c["L"], b) if "L" in c else (b,)
    if c["op"] == "evict":
        s["k"], s["v"] = _normal(g, *lead, kv, cap, d, dtype=t), _normal(g, *lead, kv, cap, d, dtype=t)
        # Sums of softmax weights: a few heavy tokens, a long tail, exact ties.
        s["mass"] = torch.exp(_normal(g, *lead, kv, cap, std=2.0))
        s["mass"] = torch.where(s["mass"] < 0.2, torch.floor(s["mass"] * 64) / 64, s["mass"])
        s["pos"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(*lead, kv, cap).contiguous()
        s["next_pos"] = s["lens"].clone()
        s["mass_out"], s["pos_out"], s["lens_out"] = torch.zeros_like(s["mass"]), torch.zeros_like(s["pos"]), torch.zeros_like(s["lens"])
        return s
    n = c["N"]
    if c["evicted"]:
        s["pos"], s["next_pos"] = _evicted_positions(g, (*lead, kv, cap), s["lens"])
    else:
        s["pos"] = s["next_pos"] = None
    if c["op"] != "tree":
        # An accepted path: increasing node numbers, ended by -1; lengths 0 .. path.
        p = c["path"]
        order = torch.rand(b, n, generator=g, device="cuda").argsort(1)[:, :p].sort(1).values.to(torch.int32)
        count = _uniform_int(g, 0, p, b)
        s["path"] = torch.where(torch.arange(p, device="cuda") < count[:, None], order, -1).to(torch.int32)
    if c["op"] == "commit":
        s["k_new"], s["v_new"] = _normal(g, *lead, kv, n, d, dtype=t), _normal(g, *lead, kv, n, d, dtype=t)
        s["k"], s["v"] = torch.zeros(*lead, kv, cap, d, device="cuda", dtype=t), torch.zeros(*lead, kv, cap, d, device="cuda", dtype=t)
        s["lens_out"], s["next_pos_out"] = torch.zeros_like(s["lens"]), torch.zeros_like(s["lens"])
        return s
    h = c["H"]
    # T5 attention has no score scale (1.0) and weights that make scores of order
    # one; the grouped-head form divides by sqrt(d).
    s["scale"] = 1.0 if d == 64 else 1.0 / math.sqrt(d)
    std = 1.5 / math.sqrt(d) / s["scale"]
    s["k"], s["v"] = _normal(g, *lead, kv, cap, d, dtype=t), _normal(g, *lead, kv, cap, d, dtype=t)
    s["rel_bias"] = _normal(g, h, c["bias"]) if c["bias"] else None
    if c["op"] == "mass":
        s["q"], s["k_new"] = _normal(g, *lead, h, n, d, std=std, dtype=t), _normal(g, *lead, kv, n, d, dtype=t)
        # Statistics of rows whose scores are of order one over the whole cache.
        s["lse"] = (s["lens"].float() + n).log()[:, None, None] + 1.0 + _normal(g, *lead, h, n, std=0.3)
        s["mass"] = torch.rand(*lead, kv, cap, generator=g, device="cuda") * 4
        s["mass_out"] = torch.zeros_like(s["mass"])
        return s
    if c["packed"]:  # the rows of one q|k|v projection
        rows = _normal(g, b, n, (h + 2 * kv) * d, dtype=t)
        rows[..., : h * d] *= std
        heads = rows.view(b, n, h + 2 * kv, d).transpose(1, 2)
        s["q"], s["k_new"], s["v_new"] = heads[:, :h], heads[:, h : h + kv], heads[:, h + kv :]
    else:
        s["q"] = _normal(g, b, h, n, d, std=std, dtype=t)
        s["k_new"], s["v_new"] = _normal(g, b, kv, n, d, dtype=t), _normal(g, b, kv, n, d, dtype=t)
    # A drafted tree: node i hangs below one of the nodes before it or below the
    # last cached token (-1); padded nodes (-2) at the end of some sequences.
    at = torch.arange(n, device="cuda")
    parents = (torch.rand(b, n, generator=g, device="cuda").sqrt() * (at + 1)).floor().clamp_(max=at) - 1
    real = n - (torch.rand(b, 1, generator=g, device="cuda") * c["pad"] * n).floor()
    s["parents"] = torch.where(at < real, parents, -2.0).to(torch.int32)
    return s


# ---- plain forms ---------------------------------------------------------------
def _seen(parents):
    """(seen[b, i, j]: node j is node i or an ancestor; absent[b, i])."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    eye = torch.eye(n, device=parents.device)
    step = eye + (parents[..., None] == at).float()
    seen = torch.matrix_power(step, max(1, n)) > 0
    wrong = (parents < -1) | (parents >= at)
    absent = (seen & wrong[:, None, :]).any(2)
    return seen & ~absent[:, :, None], absent


def _bias(table, dist, kv):
    """table (h, r) at the clamped distances dist (..., kv or 1, n, t) -> (..., kv, g, n, t)."""
    h, r = table.shape
    d = dist.clamp(0, r - 1).long().unsqueeze(-3)
    head = torch.arange(h, device=table.device).view(kv, h // kv, 1, 1)
    return table[head, d]


def _plain_tree(s):
    c, q, k_new = s["c"], s["q"], s["k_new"]
    b, h, n, d = q.shape
    kv, cap = c["KV"], c["cap"]
    seen, absent = _seen(s["parents"])
    keys = torch.cat([s["k"], k_new], 2).float()
    vals = torch.cat([s["v"], s["v_new"]], 2).float()
    at = torch.arange(cap, device=q.device)
    cached = (at < s["lens"][:, None])[:, None, :].expand(b, n, cap)
    mask = (torch.cat([cached, seen], 2) & ~absent[:, :, None])[:, None, None]
    vals = vals * (mask[:, :, 0].any(2)[..., None])
    x = (q.float().reshape(b, kv, -1, d) @ keys.transpose(2, 3)).view(b, kv, h // kv, n, cap + n) * s["scale"]
    if s["rel_bias"] is not None:
        depth = seen.sum(2) - 1
        base = s["lens"] if s["next_pos"] is None else s["next_pos"]
        pos = at.expand(b, 1, cap) if s["pos"] is None else s["pos"]
        old = (base[:, None] + depth)[:, None, :, None] - pos[:, :, None, :]
        new = (depth[:, :, None] - depth[:, None, :])[:, None].expand(b, old.shape[1], n, n)
        x = x + _bias(s["rel_bias"], torch.cat([old, new], 3), kv)
    x = torch.where(mask, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = (e.view(b, kv, -1, cap + n) @ vals).view(b, kv, h // kv, n, d) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return out.view(b, h, n, d).to(q.dtype), lse.view(b, h, n)


def _path_length(path, lens, cap):
    """Nodes of each path: up to the first negative entry, as many as fit."""
    return torch.minimum((path >= 0).long().cumprod(1).sum(1), (cap - lens).long())


def _plain_mass(s):
    c, q = s["c"], s["q"]
    L, b, h, n, d = q.shape
    kv, cap, p = c["KV"], c["cap"], s["path"].shape[1]
    count = _path_length(s["path"], s["lens"], cap)
    node = s["path"].clamp(min=0).long()[None, :, None, :]
    rows = torch.gather(q, 3, node[..., None].expand(L, b, h, p, d)).float().view(L, b, kv, h // kv, p, d)
    lse = torch.gather(s["lse"], 3, node.expand(L, b, h, p)).view(L, b, kv, h // kv, p, 1)
    new = torch.gather(s["k_new"], 3, node[..., None].expand(L, b, kv, p, d))
    keys = torch.cat([s["k"], new], 3).float()
    x = (rows.view(L, b, kv, -1, d) @ keys.transpose(3, 4)).view(L, b, kv, h // kv, p, cap + p) * s["scale"]
    at, on = torch.arange(cap, device=q.device), torch.arange(p, device=q.device)
    if s["rel_bias"] is not None:
        base = s["lens"] if s["next_pos"] is None else s["next_pos"]
        pos = at.expand(L, b, 1, cap) if s["pos"] is None else s["pos"]
        old = (base[:, None] + on)[None, :, None, :, None] - pos[:, :, :, None, :]
        step = (on[:, None] - on).expand(L, b, old.shape[2], p, p)
        x = x + _bias(s["rel_bias"], torch.cat([old, step], 4), kv)
    row = (on < count[:, None])[:, None, None, :, None]
    see = torch.cat([(at < s["lens"][:, None])[:, None, :].expand(b, p, cap), (on[:, None] >= on).expand(b, p, p)], 2)
    w = torch.where(row & see[:, None, None], torch.exp(x - lse), 0.0).sum((3, 4))
    old = at < s["lens"][:, None, None]
    out = s["mass_out"]
    slot = s["lens"][:, None] + on
    fits = on < count[:, None]
    moved = torch.zeros(L, b, kv, cap + p, device=q.device)
    moved.scatter_(3, torch.where(fits, slot, cap + on)[None, :, None].expand(L, b, kv, p).long(), w[..., cap:])
    fresh = (at >= s["lens"][:, None, None]) & (at < (s["lens"] + count)[:, None, None])
    out.copy_(torch.where(old, s["mass"] + w[..., :cap], torch.where(fresh, moved[..., :cap], out)))
    return out


def _plain_commit(s):
    c = s["c"]
    L, b, kv, n, d = s["k_new"].shape
    cap = c["cap"]
    count = _path_length(s["path"], s["lens"], cap)
    on = torch.arange(cap, device="cuda") - s["lens"][:, None]
    new = (on >= 0) & (on < count[:, None])
    node = torch.gather(s["path"].long(), 1, on.clamp(0, s["path"].shape[1] - 1).long()).clamp(min=0)
    at = new.nonzero()
    src = node[at[:, 0], at[:, 1]]
    s["k"][:, at[:, 0], :, at[:, 1]] = s["k_new"][:, at[:, 0], :, src]
    s["v"][:, at[:, 0], :, at[:, 1]] = s["v_new"][:, at[:, 0], :, src]
    s["lens_out"].copy_(s["lens"] + count)
    if s["pos"] is None:
        return s["k"], s["v"], s["lens_out"]
    s["pos"].copy_(torch.where(new[:, None], (s["next_pos"][:, None] + on)[:, None], s["pos"]))
    s["next_pos_out"].copy_(s["next_pos"] + count)
    return s["k"], s["v"], s["pos"], s["lens_out"], s["next_pos_out"]


def _plain_evict(s):
    c = s["c"]
    cap, budget = c["cap"], min(c["budget"], c["cap"])
    at = torch.arange(cap, device="cuda")
    used = (at < s["lens"][:, None, None]).expand_as(s["pos"])
    safe = (s["pos"] >= (s["next_pos"] - c["recent"])[:, None, None]) | (s["pos"] < c["sinks"])
    bits = (s["mass"] + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -2147483648 - bits)
    key = torch.where(torch.isnan(s["mass"]), -(1 << 40), key)
    key = torch.where(used, torch.where(safe, 1 << 40, key), -(1 << 41))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    kept = used & (rank < budget)
    hole, fill = used & ~kept & (at < budget), kept & (at >= budget)
    # The i-th hole below the budget takes the i-th kept row above it.
    by_rank = torch.zeros_like(order)
    spare = torch.full_like(order, cap - 1)
    first = torch.where(fill, fill.long().cumsum(-1) - 1, spare)
    by_rank.scatter_(-1, first, torch.where(fill, at, 0).expand_as(order))
    src = torch.where(hole, torch.gather(by_rank, -1, (hole.long().cumsum(-1) - 1).clamp(min=0)), at.expand_as(order))[..., :budget]
    rows = src[..., None].expand(*src.shape, c["D"])
    s["k"][..., :budget, :] = torch.gather(s["k"], 3, rows)
    s["v"][..., :budget, :] = torch.gather(s["v"], 3, rows)
    keep = used[..., :budget]
    s["mass_out"][..., :budget] = torch.where(keep, torch.gather(s["mass"], 3, src), s["mass_out"][..., :budget])
    s["pos_out"][..., :budget] = torch.where(keep, torch.gather(s["pos"], 3, src), s["pos_out"][..., :budget])
    s["lens_out"].copy_(s["lens"].clamp(max=budget))
    return s["k"], s["v"], s["mass_out"], s["pos_out"], s["lens_out"]


def _plain_q4(s):
    c = s["c"]
    p = s["packed"]
    w = torch.stack([p & 15, p >> 4], 2).view(c["N"], -1, c["group"]).float()
    w = (w * s["scales"].float()[..., None] + s["biases"].float()[..., None]).view(c["N"], c["K"])
    return (s["x"].float() @ w.t()).to(TYPES[c["out"]])


def _own(s):
    m, c = _ops(), s["c"]
    if c["op"] == "tree":
        return m.tree_attention(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["lens"], s["parents"], scale=s["scale"],
                                rel_bias=s["rel_bias"], pos=s["pos"], next_pos=s["next_pos"])
    if c["op"] == "mass":
        return m.cache_mass(s["q"], s["lse"], s["k_new"], s["k"], s["lens"], s["path"], s["mass"], scale=s["scale"],
                            rel_bias=s["rel_bias"], pos=s["pos"], next_pos=s["next_pos"], mass_out=s["mass_out"])
    if c["op"] == "commit":
        m.cache_commit(s["k_new"], s["v_new"], s["k"], s["v"], s["lens"], s["path"], pos=s["pos"], next_pos=s["next_pos"],
                       lens_out=s["lens_out"], next_pos_out=None if s["pos"] is None else s["next_pos_out"])
        if s["pos"] is None:
            return s["k"], s["v"], s["lens_out"]
        return s["k"], s["v"], s["pos"], s["lens_out"], s["next_pos_out"]
    if c["op"] == "evict":
        m.cache_evict(s["k"], s["v"], s["lens"], s["mass"], s["pos"], s["next_pos"], budget=c["budget"], recent=c["recent"],
                      sinks=c["sinks"], mass_out=s["mass_out"], pos_out=s["pos_out"], lens_out=s["lens_out"])
        return s["k"], s["v"], s["mass_out"], s["pos_out"], s["lens_out"]
    return m.q4_linear(s["x"], s["packed"], s["scales"], s["biases"], out_dtype=TYPES[c["out"]])


PLAIN = {"tree": _plain_tree, "mass": _plain_mass, "commit": _plain_commit, "evict": _plain_evict, "q4": _plain_q4}


def run(s):
    if own:
        return _own(s)
    return PLAIN[s["c"]["op"]](s)


# ---- 64-bit values ---------------------------------------------------------------
def _ancestors(parents):
    """Per sequence and node: its chain from the root to itself, or None if absent."""
    chains = []
    for row in parents:
        mine = []
        for i, p in enumerate(row):
            if p == -1:
                mine.append([i])
            elif 0 <= p < i and mine[p] is not None:
                mine.append(mine[p] + [i])
            else:
                mine.append(None)
        chains.append(mine)
    return chains


def _exact_tree(c, s):
    b, h, n, d = s["q"].shape
    kv, dev = c["KV"], s["q"].device
    grp = h // kv
    out = torch.zeros(b, h, n, d, dtype=torch.float64, device=dev)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=dev)
    chains = _ancestors(s["parents"].cpu().tolist())
    for i in range(b):
        t = int(s["lens"][i])
        q = s["q"][i].double().reshape(kv, grp, n, d)
        x = torch.einsum("kgnd,ktd->kgnt", q, s["k"][i, :, :t].double()) * s["scale"]
        y = torch.einsum("kgnd,kjd->kgnj", q, s["k_new"][i].double()) * s["scale"]
        vis = np.zeros((n, n), bool)
        depth = np.zeros(n, np.int64)
        for a, chain in enumerate(chains[i]):
            if chain is not None:
                vis[a, chain] = True
                depth[a] = len(chain) - 1
        dep = torch.from_numpy(depth).to(dev)
        there = torch.from_numpy(vis.any(1)).to(dev)
        if s["rel_bias"] is not None:
            tab = s["rel_bias"].double().view(kv, grp, -1)
            r = tab.shape[2]
            start = t if s["next_pos"] is None else int(s["next_pos"][i])
            where = torch.arange(t, device=dev).expand(kv, t) if s["pos"] is None else s["pos"][i, :, :t].long()
            far = (start + dep)[None, :, None] - where[:, None, :]
            for k in range(kv):
                x[k] += tab[k][:, far[k].clamp(0, r - 1)]
            y += tab[:, :, (dep[:, None] - dep[None, :]).clamp(0, r - 1)]
        y = y.masked_fill(~torch.from_numpy(vis).to(dev), -math.inf)
        z = torch.cat([x, y], 3)[:, :, there]
        if z.shape[2]:
            total = torch.logsumexp(z, 3)
            w = torch.exp(z - total[..., None])
            v = torch.cat([s["v"][i, :, :t], s["v_new"][i]], 1).double()
            out[i].view(kv, grp, n, d)[:, :, there] = torch.einsum("kgnt,ktd->kgnd", w, v)
            lse[i].view(kv, grp, n)[:, :, there] = total
    return out, lse


def _exact_mass(c, s):
    L, b, h, n, d = s["q"].shape
    kv = c["KV"]
    grp, out = h // kv, s["mass_out"].double()
    paths = s["path"].cpu().tolist()
    for i in range(b):
        t = int(s["lens"][i])
        nodes = [x for x in paths[i] if x >= 0][: c["cap"] - t]
        a = len(nodes)
        start = t if s["next_pos"] is None else int(s["next_pos"][i])
        for j in range(L):
            keys = torch.cat([s["k"][j, i, :, :t], s["k_new"][j, i][:, nodes]], 1).double()
            for k in range(kv):
                heads = slice(k * grp, (k + 1) * grp)
                x = s["q"][j, i, heads][:, nodes].double() @ keys[k].t() * s["scale"]
                if s["rel_bias"] is not None and a:
                    where = torch.arange(t, device="cuda") if s["pos"] is None else s["pos"][j, i, k, :t].long()
                    here = start + torch.arange(a, device="cuda")
                    far = here[:, None] - torch.cat([where, here])[None]
                    x += s["rel_bias"].double()[heads][:, far.clamp(0, c["bias"] - 1)]
                w = torch.exp(x - s["lse"][j, i, heads][:, nodes].double()[..., None])
                for r in range(a):
                    w[:, r, t + r + 1 :] = 0
                w = w.sum((0, 1))
                out[j, i, k, :t] = s["mass"][j, i, k, :t].double() + w[:t]
                out[j, i, k, t : t + a] = w[t:]
    return out


def exact(c, seed):
    if c["op"] in ("commit", "evict"):
        return None  # rows are moved, nothing is computed
    s = prepare(c, seed)
    if c["op"] == "tree":
        return _exact_tree(c, s)
    if c["op"] == "mass":
        return _exact_mass(c, s)
    nib = s["packed"].cpu().numpy()
    n, k, gr = c["N"], c["K"], c["group"]
    vals = np.empty((n, k), np.uint8)
    vals[:, 0::2], vals[:, 1::2] = nib & 15, nib >> 4
    y = torch.zeros(c["M"], n, dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for a in range(0, n, 2048):
        w = torch.from_numpy(vals[a : a + 2048]).to("cuda").double()
        sc = s["scales"][a : a + 2048].double().repeat_interleave(gr, 1)
        bi = s["biases"][a : a + 2048].double().repeat_interleave(gr, 1)
        y[:, a : a + 2048] = x @ (w * sc + bi).t()
    return y
