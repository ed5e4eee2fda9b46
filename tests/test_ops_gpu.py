"""The operators on device buffers (mrtops.py) against plain 64-bit
restatements of their formulas, at the sizes, lengths and masks where they can
go wrong.

Tolerances. u is half a step of the result's type (eps / 2). A float32 sum of n
terms is off by at most n 2^-24 of the sum of absolute values when it is
sequential; the kernels' sums are split over lanes, so n / 8 + 64 terms follow
one another, and the matrix instructions round towards zero (2^-23 a step).
A score's error e is (D + 4) 2^-23 of sum |q k| |scale| (plus the bias), a
weight's relative error 2 e, the two-part bf16 weights add 2^-16."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops(mrtdf):
    import mrtops

    mrtops.lib()
    return mrtops


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- oracles ---------------------------------------------------------------------
def chains(parents, n):
    """Per node its chain from the root, None for an absent one."""
    out = []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p] is not None:
            out.append(out[p] + [i])
        else:
            out.append(None)
    return out


def attend(q, kn, vn, k, v, lens, parents=None, scale=1.0, rel_bias=None, pos=None, next_pos=None):
    """(out, lse, tolerance of out, tolerance of lse) in float64 on the CPU."""
    dt = q.dtype
    q, kn, vn, k, v = (t.detach().cpu().double() for t in (q, kn, vn, k, v))
    B, H, N, D = q.shape
    KV, cap = k.shape[1], k.shape[2]
    G = H // KV
    out, lse = torch.zeros(B, H, N, D, dtype=torch.float64), torch.full((B, H, N), -math.inf, dtype=torch.float64)
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    table = None if rel_bias is None else rel_bias.cpu().double()
    for b in range(B):
        t = int(lens[b])
        if not 0 <= t <= cap:
            continue
        ch = chains(None if parents is None else parents[b].cpu(), N)
        nxt = t if next_pos is None else int(next_pos[b])
        for h in range(H):
            g = h // G
            where = torch.arange(t) if pos is None else pos[b, g, :t].cpu().long()
            for i in range(N):
                if ch[i] is None:
                    continue
                keys, vals = torch.cat([k[b, g, :t], kn[b, g][ch[i]]]), torch.cat([v[b, g, :t], vn[b, g][ch[i]]])
                x = keys @ q[b, h, i] * scale
                mag = float((keys.abs() @ q[b, h, i].abs()).max()) * abs(scale)
                if table is not None:
                    at = torch.cat([where, nxt + torch.arange(len(ch[i]))])
                    add = table[h][(nxt + len(ch[i]) - 1 - at).clamp(0, table.shape[1] - 1)]
                    x = x + add
                    fin = add[add.abs() < 1e30]
                    mag += float(fin.abs().max()) if len(fin) else 0.0
                if not bool((x > -math.inf).any()):
                    continue
                lse[b, h, i] = torch.logsumexp(x, 0)
                w = torch.exp(x - lse[b, h, i])
                out[b, h, i] = w @ vals
                e = (D + 4) * 2.0**-23 * mag
                steps = (len(x) / 8 + 64) * 2.0**-23
                size = w @ vals.abs()
                tol[b, h, i] = half_step(dt) * out[b, h, i].abs() + size * ((2.0**-16 if dt == BF else 2.0**-20) + 4 * e + 2 * steps)
                tol_l[b, h, i] = e + steps + 2.0**-22 * (1 + abs(float(lse[b, h, i])))
    return out, lse, tol, tol_l


def collected(q, lse, kn, k, lens, path, mass, mass_out, scale=1.0, rel_bias=None, pos=None, next_pos=None, decay=1.0,
              nodes=64):
    """(mass_out, tolerance) in float64; five-dimensional inputs."""
    L, B, H, N, D = q.shape
    KV, cap = k.shape[2], k.shape[3]
    G = H // KV
    want, tol = mass_out.cpu().double().clone(), torch.zeros(mass_out.shape, dtype=torch.float64)
    q, kn, k, lse, mass = (t.cpu().double() for t in (q, kn, k, lse, mass))
    for b in range(B):
        t = int(lens[b])
        if not 0 <= t <= cap:
            continue
        mine = taken(path[b].cpu().tolist(), N, cap - t)
        a = len(mine)
        nxt = t if next_pos is None else int(next_pos[b])
        for l in range(L):
            for g in range(KV):
                keys = torch.cat([k[l, b, g, :t], kn[l, b, g][mine]])
                where = torch.arange(t) if pos is None else pos[l, b, g, :t].cpu().long()
                where = torch.cat([where, nxt + torch.arange(a)])
                total, err = torch.zeros(t + a, dtype=torch.float64), torch.zeros(t + a, dtype=torch.float64)
                for h in range(g * G, (g + 1) * G):
                    for r, n in enumerate(mine):
                        if lse[l, b, h, n] == -math.inf:
                            continue
                        x = keys @ q[l, b, h, n] * scale
                        mag = keys.abs() @ q[l, b, h, n].abs() * abs(scale)
                        if rel_bias is not None:
                            add = rel_bias.cpu().double()[h][(nxt + r - where).clamp(0, rel_bias.shape[1] - 1)]
                            x, mag = x + add, mag + add.abs()
                        w = torch.exp(x - lse[l, b, h, n])
                        w[t + r + 1:] = 0
                        total += w
                        err += w * (2 * (D + 4) * 2.0**-23 * mag + 2.0**-20 + 2.0**-22 * (x - lse[l, b, h, n]).abs())
                total[:t] += decay * mass[l, b, g, :t]
                want[l, b, g, : t + a] = total
                tol[l, b, g, : t + a] = err + total.abs() * (a * G + 8) * 2.0**-23
    return want, tol


def taken(path, nodes, room):
    """The accepted nodes: increasing, inside [0, nodes), as many as fit."""
    out = []
    for n in path:
        if not 0 <= n < nodes or (out and n <= out[-1]):
            break
        out.append(n)
    return out[: max(0, room)]


def near(got, want, tol):
    got = got.detach().cpu().double()
    same = (got == want) | ((got - want).abs() <= tol)
    bad = ~same
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} values off, the worst {float(((got - want).abs() / tol.clamp(min=1e-300))[bad].max()):.3g} "
        f"tolerances; first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])}")


def normal(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def tree_of(rng, n, pad=0):
    p = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
    for i in range(n - pad, n):
        p[i] = int(rng.choice([-2, i, 99, -2147483648, 2147483647]))
    return p


def tree_inputs(seed, dtype, B, H, KV, N, D, cap, std=None):
    std = 1.5 / math.sqrt(D) if std is None else std
    return (normal(seed, B, H, N, D, dtype=dtype, std=std), normal(seed + 1, B, KV, N, D, dtype=dtype),
            normal(seed + 2, B, KV, N, D, dtype=dtype), normal(seed + 3, B, KV, cap, D, dtype=dtype),
            normal(seed + 4, B, KV, cap, D, dtype=dtype))


def check_tree(ops, inputs, lens, parents, **kw):
    out, lse = ops.tree_attention(*inputs, lens, parents, **kw)
    wo, wl, to, tl = attend(*inputs, lens, parents, **{k: v for k, v in kw.items() if k not in ("out", "lse", "workspace")})
    near(out, wo, to)
    near(lse, wl, tl)
    return out, lse


# ---- tree attention ----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV,N", [(2, 2, 1), (4, 4, 16), (3, 1, 5), (8, 2, 8), (4, 2, 24), (2, 1, 33), (2, 2, 64), (8, 1, 17)])
def test_tree_sizes(ops, dtype, D, H, KV, N):
    rng = np.random.default_rng(N * 7 + D)
    cap = 200
    lens = [0, 1, 63, 64, 200, 137]
    parents = ints([tree_of(rng, N, N // 5 if b == 5 else 0) for b in range(6)])
    check_tree(ops, tree_inputs(N, dtype, 6, H, KV, N, D, cap), ints(lens), parents)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,KV,N,cap,lens", [
    (1, 1, 1, 1, 6000, [5999]), (1, 2, 1, 16, 5000, [5000]), (3, 4, 2, 12, 1300, [1300, 0, 650]),
    (2, 2, 2, 40, 700, [64 * 10 - 40, 641]), (5, 1, 1, 2, 400, [400, 399, 1, 255, 256])])
def test_tree_split_over_ctas(ops, dtype, B, H, KV, N, cap, lens):
    rng = np.random.default_rng(cap)
    parents = ints([tree_of(rng, N) for _ in range(B)])
    check_tree(ops, tree_inputs(cap, dtype, B, H, KV, N, 64, cap), ints(lens), parents)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap,rel_len", [(100, 128), (100, 16), (900, 128), (900, 1)])
@pytest.mark.parametrize("stored", [False, True])
def test_tree_relative_bias(ops, dtype, cap, rel_len, stored):
    B, H, KV, N = 3, 4, 2, 9
    rng = np.random.default_rng(cap + rel_len)
    lens = ints([cap, 7, cap // 2])
    kw = dict(rel_bias=normal(9, H, rel_len))
    if stored:
        pos = torch.stack([torch.stack([torch.from_numpy(rng.permutation(3 * cap)[:cap]) for _ in range(KV)]) for _ in range(B)])
        kw |= dict(pos=pos.to(torch.int32).to(DEV).contiguous(), next_pos=ints([3 * cap, 3 * cap + 5, 3 * cap + 1]))
    parents = ints([tree_of(rng, N, 2) for _ in range(B)])
    check_tree(ops, tree_inputs(cap, dtype, B, H, KV, N, 64, cap), lens, parents, **kw)


@pytest.mark.parametrize("N", [1, 7, 64])
def test_tree_without_parents_is_a_chain(ops, N):
    x = tree_inputs(N, F32, 2, 2, 2, N, 64, 90)
    lens = ints([90, 3])
    a = check_tree(ops, x, lens, None)
    b = ops.tree_attention(*x, lens, ints([list(range(-1, N - 1))] * 2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [80, 500])
def test_tree_lengths_that_make_no_sense_give_empty_rows(ops, dtype, cap):
    x = tree_inputs(3, dtype, 4, 2, 1, 5, 64, cap)
    lens = ints([-1, cap + 1, -2147483648, cap])
    out, lse = check_tree(ops, x, lens, None)
    assert not out[:3].any() and bool((lse[:3] == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [80, 500])
def test_tree_values_that_are_not_seen_do_not_matter(ops, dtype, cap):
    """NaN and infinities behind the length, in absent nodes, and in a branch
    that the other branch does not see."""
    q, kn, vn, k, v = tree_inputs(5, dtype, 2, 2, 2, 6, 64, cap)
    lens = ints([cap - 30, 0])
    for b in range(2):
        for t, fill in ((k, math.nan), (v, math.inf)):
            t[b, :, int(lens[b]):] = fill
    parents = ints([[-1, 0, -1, 2, -2, 4]] * 2)  # two chains (0, 1), (2, 3); 4 and 5 absent
    kn[:, :, 4:], vn[:, :, 4:], q[:, :, 4:] = math.nan, -math.inf, math.nan
    kn[:, :, 3], vn[:, :, 3] = math.nan, math.nan
    out, lse = ops.tree_attention(q, kn, vn, k, v, lens, parents)
    zero = [t.clone() for t in (q, kn, vn, k, v)]
    for t in zero:
        t[~torch.isfinite(t)] = 0
    wo, wl, to, tl = attend(*zero, lens, parents)
    for n in (0, 1, 2, 4, 5):
        near(out[:, :, n], wo[:, :, n], to[:, :, n])
        near(lse[:, :, n], wl[:, :, n], tl[:, :, n])
    assert bool(torch.isnan(out[:, :, 3]).all())


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(F32).min])
@pytest.mark.parametrize("cap", [100, 600])
def test_tree_bias_of_the_lowest_value(ops, low, cap):
    """-inf everywhere leaves a row empty; the lowest number everywhere is a
    constant (softmax over what the scores add to it)."""
    x = tree_inputs(6, F32, 2, 2, 2, 3, 64, cap)
    lens = ints([cap, 40])
    bias = torch.full((2, 32), low, device=DEV)
    out, lse = ops.tree_attention(*x, lens, None, rel_bias=bias)
    if low == -math.inf:
        assert not out.any() and bool((lse == -math.inf).all())
        bias[:, 31] = 0.0  # only far rows are left
        check_tree(ops, x, lens, None, rel_bias=bias)
    else:  # every score rounds to the lowest number: equal weights
        k, v = torch.cat([x[3], x[1]], 2), torch.cat([x[4], x[2]], 2)
        for b, t in enumerate(lens.tolist()):
            for i in range(3):
                vals = torch.cat([x[4][b, :, :t], x[2][b, :, : i + 1]], 1).cpu().double()
                near(out[b, :, i], vals.mean(1), 2.0**-14 * vals.abs().mean(1))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [120, 700])
def test_tree_strided_views(ops, dtype, cap):
    """q, k, v as views of one projection, a cache with the heads inside the
    rows, an output view; what lies between the views stays as it was."""
    B, H, KV, N, D = 2, 4, 2, 6, 64
    rows = normal(1, B, N, (H + 2 * KV) * D, dtype=dtype, std=0.3).view(B, N, H + 2 * KV, D).transpose(1, 2)
    q, kn, vn = rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:]
    both = normal(2, B, cap, 2, KV, D, dtype=dtype)
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    base = torch.full((B, N, H + 1, D), 7.0, dtype=dtype, device=DEV)
    out = base[:, :, :H].transpose(1, 2)
    check_tree(ops, (q, kn, vn, k, v), ints([cap, 33]), None, out=out)
    assert bool((base[:, :, H] == 7).all())


def test_tree_large_scores(ops):
    """Scores of some hundreds: the running maximum rises tile by tile."""
    x = list(tree_inputs(8, F32, 1, 2, 2, 4, 64, 900, std=1.0))
    x[3] *= torch.linspace(0.1, 12, 900, device=DEV)[None, None, :, None]
    check_tree(ops, x, ints([900]), None)


def test_tree_is_the_same_every_time_and_on_any_stream(ops):
    x = tree_inputs(9, BF, 3, 8, 2, 12, 128, 1500)
    lens = ints([1500, 3, 800])
    first = ops.tree_attention(*x, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.tree_attention(*x, lens)
    other = ops.tree_attention(*x, lens)
    torch.cuda.synchronize()
    for r in (again, other):
        assert torch.equal(first[0], r[0]) and torch.equal(first[1], r[1])


def test_tree_captured_twice_and_replayed_at_once(ops):
    """Two captured graphs have workspaces of their own; lengths are read when
    the graph runs."""
    x = tree_inputs(10, BF, 2, 4, 2, 8, 64, 2000)
    lens = ints([2000, 70])
    ops.tree_attention(*x, lens)
    pairs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.tree_attention(*x, lens)
        pairs.append((g, r, torch.cuda.Stream()))
    for now in ([2000, 70], [5, 1999]):
        lens.copy_(ints(now))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, s in pairs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        wo, wl, to, tl = attend(*x, lens)
        for _, r, _ in pairs:
            near(r[0], wo, to)
            near(r[1], wl, tl)


def test_tree_cache_past_32_bits(ops):
    """Rows beyond element 2^31 of the cache."""
    B, KV, cap, D = 5, 4, 1 << 20, 128
    k = torch.empty(B, KV, cap, D, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    assert k.numel() > 2**31
    small = tree_inputs(11, BF, 1, 4, 4, 3, D, 300)
    k[4, :, :300], v[4, :, :300] = small[3][0], small[4][0]
    q, kn, vn = (t.expand(5, -1, -1, -1).contiguous() for t in small[:3])
    out, lse = ops.tree_attention(q, kn, vn, k, v, ints([0, 0, 0, 0, 300]))
    wo, wl, to, tl = attend(*small, ints([300]))
    near(out[4:], wo, to)
    near(lse[4:], wl, tl)
    # the last rows of the last head, behind a cache whose other rows are far away
    k[4, 3, -200:], v[4, 3, -200:] = small[3][0, 3, :200], small[4][0, 3, :200]
    tail_k, tail_v = k[4:, 3:, -200:], v[4:, 3:, -200:]
    out, lse = ops.tree_attention(small[0][:, 3:], small[1][:, 3:], small[2][:, 3:], tail_k, tail_v, ints([200]))
    wo, wl, to, tl = attend(small[0][:, 3:], small[1][:, 3:], small[2][:, 3:], tail_k, tail_v, ints([200]))
    near(out, wo, to)


def test_tree_many_sequences(ops):
    B = 1024
    x = tree_inputs(12, BF, B, 1, 1, 2, 64, 70)
    lens = torch.arange(B, device=DEV, dtype=torch.int32) % 72 - 1  # -1 and 70 among them
    out, lse = ops.tree_attention(*x, lens)
    pick = [0, 1, 2, 71, 72, 500, 1023]
    wo, wl, to, tl = attend(*(t[pick] for t in x), lens[pick])
    near(out[pick], wo, to)
    near(lse[pick], wl, tl)


def test_tree_refuses(ops, mrtdf):
    q, kn, vn, k, v = x = tree_inputs(1, BF, 2, 4, 2, 3, 64, 50)
    lens = ints([1, 2])
    bad = [
        lambda: ops.tree_attention(q.float(), kn, vn, k, v, lens),
        lambda: ops.tree_attention(q[:, :3], kn, vn, k, v, lens),
        lambda: ops.tree_attention(*x, lens.long()),
        lambda: ops.tree_attention(*x, lens.cpu()),
        lambda: ops.tree_attention(*x, lens[:1]),
        lambda: ops.tree_attention(*(t[..., :32] for t in x), lens),
        lambda: ops.tree_attention(q, kn, vn, k, v[:, :, :49], lens),
        lambda: ops.tree_attention(q, kn, vn, k.transpose(2, 3), v.transpose(2, 3), lens),
        lambda: ops.tree_attention(*x, lens, ints([[0, 0]])),
        lambda: ops.tree_attention(*x, lens, rel_bias=torch.zeros(3, 8, device=DEV)),
        lambda: ops.tree_attention(*x, lens, pos=torch.zeros(2, 2, 50, dtype=torch.int32, device=DEV)),
        lambda: ops.tree_attention(*x, lens, scale=math.nan),
        lambda: ops.tree_attention(q.clone().requires_grad_(), kn, vn, k, v, lens),
        lambda: ops.tree_attention(*(t.half() for t in x), lens),
        lambda: ops.tree_attention(*tree_inputs(1, BF, 2, 1, 1, 3, 64, 600), lens,
                                   workspace=torch.empty(16, dtype=torch.uint8, device=DEV)),
        lambda: ops.tree_attention(*tree_inputs(1, BF, 2, 1, 1, 65, 64, 8), lens),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(mrtdf.MrtdfError) as e:
            f()
        assert e.value.code in (1, 7), i
    # an odd element offset: rows that do not start on 16 bytes
    odd = torch.zeros(2 * 4 * 3 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, 4, 3, 64)
    with pytest.raises(mrtdf.MrtdfError, match="16-byte"):
        ops.tree_attention(odd, kn, vn, k, v, lens)
    check_tree(ops, x, lens, None)  # nothing is left behind


# ---- collected weight -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L,H,KV,N,P,cap", [(1, 2, 2, 1, 1, 70), (2, 4, 2, 9, 4, 300), (1, 8, 1, 24, 16, 200), (1, 2, 1, 64, 64, 130)])
@pytest.mark.parametrize("bias", [0, 32])
def test_mass(ops, dtype, D, L, H, KV, N, P, cap, bias):
    B = 5
    rng = np.random.default_rng(cap + N)
    lens = [0, cap, cap - 2, 64, -1]
    path = np.full((B, P), -1)
    for b in range(B):
        n = min(P, [P, P, P, P // 2, P][b])
        path[b, :n] = np.sort(rng.permutation(N)[:n])
    path = ints(path.tolist())
    q, k, kn = normal(1, L, B, H, N, D, dtype=dtype, std=0.2), normal(2, L, B, KV, cap, D, dtype=dtype), normal(3, L, B, KV, N, D, dtype=dtype)
    lse = normal(4, L, B, H, N) + 4
    lse[0, 1, 0, int(path[1, 0])] = -math.inf
    mass, out = normal(5, L, B, KV, cap).abs(), normal(6, L, B, KV, cap)
    kw = dict(scale=1.0, decay=0.9)
    if bias:
        pos = torch.stack([torch.from_numpy(rng.permutation(2 * cap)[:cap]) for _ in range(L * B * KV)])
        kw |= dict(rel_bias=normal(7, H, bias), pos=pos.view(L, B, KV, cap).to(torch.int32).to(DEV), next_pos=ints([2 * cap] * B))
    want, tol = collected(q, lse, kn, k, ints(lens), path, mass, out, **kw)
    got = ops.cache_mass(q, lse, kn, k, ints(lens), path, mass, mass_out=out, **kw)
    assert got is out
    near(out, want, tol)
    inplace = mass.clone()
    ops.cache_mass(q, lse, kn, k, ints(lens), path, inplace, **kw)
    for b, t in enumerate(lens):
        if t < 0:
            assert torch.equal(inplace[:, b], mass[:, b])
            continue
        a = len(taken(path[b].tolist(), N, cap - t))
        assert torch.equal(inplace[:, b, :, : t + a], out[:, b, :, : t + a])
        assert torch.equal(inplace[:, b, :, t + a:], mass[:, b, :, t + a:])


def test_mass_of_one_token_sums_to_its_heads(ops):
    """Softmax weights of one decoded token: each query head adds one."""
    B, H, KV, D, cap = 2, 6, 2, 64, 500
    q, kn, vn, k, v = tree_inputs(2, F32, B, H, KV, 1, D, cap)
    lens = ints([499, 17])
    _, lse = ops.tree_attention(q, kn, vn, k, v, lens)
    mass = torch.zeros(B, KV, cap, device=DEV)
    ops.cache_mass(q, lse, kn, k, lens, ints([[0], [0]]), mass)
    near(mass.sum(2), torch.full((B, KV), 3.0, dtype=torch.float64), torch.full((B, KV), 3 * 2.0**-13))


def test_mass_refuses(ops, mrtdf):
    q, k, kn = normal(1, 1, 2, 4, 64), normal(2, 1, 2, 20, 64), normal(3, 1, 2, 4, 64)
    lse, mass, lens, path = torch.zeros(1, 2, 4, device=DEV), torch.zeros(1, 2, 20, device=DEV), ints([3]), ints([[0, 1]])
    for f in (lambda: ops.cache_mass(q, lse, kn, k, lens, ints([[0, 1, 2, 3, 4]]), mass),
              lambda: ops.cache_mass(q, lse, kn, k, lens, path, mass[..., :19]),
              lambda: ops.cache_mass(q, lse[..., :3], kn, k, lens, path, mass),
              lambda: ops.cache_mass(q, lse, kn, k, lens, path[0], mass),
              lambda: ops.cache_mass(q, lse, kn, k, lens, path, mass, decay=math.nan),
              lambda: ops.cache_mass(q, lse, kn, k, lens, path, mass.double())):
        with pytest.raises(mrtdf.MrtdfError):
            f()


# ---- commit -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L,KV,N,P,cap", [(1, 1, 1, 1, 10), (3, 2, 9, 5, 40), (2, 4, 64, 64, 100), (1, 3, 40, 33, 90)])
def test_commit(ops, dtype, D, L, KV, N, P, cap):
    rng = np.random.default_rng(N)
    paths, lens = [], []
    for b in range(7):
        p = np.full(P, -1)
        n = [P, 0, P // 2, P, P, P, P][b]
        p[:n] = np.sort(rng.permutation(N)[:n])
        if b == 3 and P > 2:
            p[2] = p[1]  # not above the one before: the path ends
        if b == 4 and P > 1:
            p[1] = N  # no such node
        paths.append(p.tolist())
        lens.append([0, 3, cap - 1, 2, 5, cap, cap + 1][b])
    kn, vn = normal(1, L, 7, KV, N, D, dtype=dtype), normal(2, L, 7, KV, N, D, dtype=dtype)
    k, v = normal(3, L, 7, KV, cap, D, dtype=dtype), normal(4, L, 7, KV, cap, D, dtype=dtype)
    pos = torch.full((L, 7, KV, cap), -5, dtype=torch.int32, device=DEV)
    nxt = ints([100 + b for b in range(7)])
    wk, wv, wp, wl, wn = k.clone(), v.clone(), pos.clone(), list(lens), nxt.tolist()
    for b in range(7):
        if not 0 <= lens[b] <= cap:
            continue
        mine = taken(paths[b], N, cap - lens[b])
        for j, n in enumerate(mine):
            wk[:, b, :, lens[b] + j], wv[:, b, :, lens[b] + j] = kn[:, b, :, n], vn[:, b, :, n]
            wp[:, b, :, lens[b] + j] = 100 + b + j
        wl[b] += len(mine)
        wn[b] += len(mine)
    out, nout = ops.cache_commit(kn, vn, k, v, ints(lens), ints(paths), pos=pos, next_pos=nxt)
    assert out.tolist() == wl and nout.tolist() == wn
    assert torch.equal(k, wk) and torch.equal(v, wv) and torch.equal(pos, wp)


def test_commit_of_one_layer_and_views(ops):
    kn = normal(1, 2, 6, 4, 64).transpose(1, 2)  # (2, 4, 6, 64)
    both = torch.zeros(2, 30, 2, 4, 64, device=DEV)
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    lens, n = ops.cache_commit(kn, kn, k, v, ints([0, 28]), ints([[1, 3, 5], [0, 1, 2]]))
    assert lens.tolist() == [3, 30] and n is None
    assert torch.equal(k[0, :, :3], kn[0, :, [1, 3, 5]]) and torch.equal(v[1, :, 28:], kn[1, :, :2])
    assert not both[0, 3:].any() and not both[1, :28].any()


def test_commit_refuses(ops, mrtdf):
    kn, k = normal(1, 1, 2, 4, 64), normal(2, 1, 2, 20, 64)
    lens, path = ints([3]), ints([[0, 1]])
    for f in (lambda: ops.cache_commit(kn, kn, k, k, lens, path, lens_out=lens),
              lambda: ops.cache_commit(kn, kn, k, k, lens, path, next_pos_out=ints([0])),
              lambda: ops.cache_commit(kn, kn[:, :1], k, k, lens, path),
              lambda: ops.cache_commit(kn, kn, k, k, lens, ints([[0, 1, 2, 3, 3]])),
              lambda: ops.cache_commit(kn.bfloat16(), kn.bfloat16(), k, k, lens, path)):
        with pytest.raises(mrtdf.MrtdfError):
            f()


# ---- eviction ----------------------------------------------------------------------
def evicted(k, v, lens, mass, pos, next_pos, budget, recent, sinks, mass_out, pos_out):
    """In place on numpy copies; five-dimensional."""
    L, B, KV, cap = mass.shape
    out = lens.copy()
    for b in range(B):
        n = int(lens[b])
        if not 0 <= n <= cap:
            continue
        out[b] = min(n, budget)
        for l in range(L):
            for h in range(KV):
                m, p = mass[l, b, h], pos[l, b, h]
                keep = set(range(n))
                if n > budget:
                    safe = (p[:n].astype(np.int64) >= int(next_pos[b]) - recent) | (p[:n] < sinks)

                    def rank(t):
                        return (not safe[t], 0 if safe[t] else (math.inf if math.isnan(m[t]) else -float(m[t])),
                                not safe[t] and bool(math.isnan(m[t])), t)

                    keep = set(sorted(range(n), key=rank)[:budget])
                holes = [t for t in range(min(n, budget)) if t not in keep]
                fills = [t for t in sorted(keep) if t >= budget]
                m0, p0 = m.copy(), p.copy()
                for t in keep:
                    if t < budget:
                        mass_out[l, b, h, t], pos_out[l, b, h, t] = m0[t], p0[t]
                for dst, src in zip(holes, fills):
                    k[l, b, h, dst], v[l, b, h, dst] = k[l, b, h, src], v[l, b, h, src]
                    mass_out[l, b, h, dst], pos_out[l, b, h, dst] = m0[src], p0[src]
    return out


def evict_case(ops, L, B, KV, cap, D, lens, budget, recent, sinks, dtype=F32, weights=None, seed=0, apart=True):
    rng = np.random.default_rng(seed)
    mass = rng.exponential(size=(L, B, KV, cap)).astype(np.float32) if weights is None else weights
    pos = np.stack([rng.permutation(4 * cap)[:cap] for _ in range(L * B * KV)]).reshape(L, B, KV, cap).astype(np.int32)
    nxt = np.full(B, 4 * cap, np.int32)
    k, v = normal(seed, L, B, KV, cap, D, dtype=dtype), normal(seed + 1, L, B, KV, cap, D, dtype=dtype)
    kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
    dm, dp = torch.from_numpy(mass.copy()).to(DEV), torch.from_numpy(pos.copy()).to(DEV)
    mo, po = (torch.full_like(dm, -3), torch.full_like(dp, -3)) if apart else (dm, dp)
    wm, wp = mo.cpu().numpy().copy(), po.cpu().numpy().copy()
    wl = evicted(kn, vn, np.array(lens, np.int32), mass, pos, nxt, budget, recent, sinks, wm, wp)
    got = ops.cache_evict(k, v, ints(lens), dm, dp, torch.from_numpy(nxt).to(DEV), budget=budget, recent=recent, sinks=sinks,
                          mass_out=mo if apart else None, pos_out=po if apart else None)
    assert got.tolist() == wl.tolist()
    assert np.array_equal(po.cpu().numpy(), wp)
    assert np.array_equal(mo.cpu().numpy(), wm, equal_nan=True)
    assert np.array_equal(k.float().cpu().numpy(), kn) and np.array_equal(v.float().cpu().numpy(), vn)


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 128)])
@pytest.mark.parametrize("L,B,KV,cap,lens,budget,recent,sinks", [
    (1, 1, 1, 8, [8], 1, 0, 0), (2, 4, 2, 50, [50, 40, 41, 0], 40, 8, 1), (1, 3, 1, 700, [700, 699, -1], 33, 10, 4),
    (1, 2, 1, 3000, [3000, 2049], 2048, 100, 4), (1, 2, 2, 5000, [5000, 4999], 64, 64, 0), (1, 2, 1, 64, [65, 64], 63, 0, 0)])
def test_evict(ops, apart, dtype, D, L, B, KV, cap, lens, budget, recent, sinks):
    evict_case(ops, L, B, KV, cap, D, lens, budget, recent, sinks, dtype, apart=apart)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "nan", "inf"])
@pytest.mark.parametrize("cap", [300, 9000])
def test_evict_ties_and_odd_weights(ops, kind, cap):
    """Ties go to the lowest row (-0 = +0), NaN comes last."""
    rng = np.random.default_rng(cap)
    w = rng.choice([0.0, -0.0, 1.0, 2.0], size=(1, 2, 1, cap)).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "signs":
        w = rng.standard_normal(w.shape).astype(np.float32).round(1)
    elif kind == "nan":
        w[rng.random(w.shape) < 0.7] = np.nan
    elif kind == "inf":
        w[rng.random(w.shape) < 0.4] = np.inf
        w[rng.random(w.shape) < 0.4] = -np.inf
    evict_case(ops, 1, 2, 1, cap, 64, [cap, cap - 1], cap // 3, cap // 10, 2, weights=w)


def test_evict_long_cache(ops):
    """Keys that do not fit into shared memory and several rounds of moves."""
    evict_case(ops, 1, 1, 1, 150000, 64, [150000], 70000, 500, 4, BF)


def test_evict_in_graph_many_heads(ops):
    L, B, KV, cap, D = 4, 8, 8, 130, 64
    k, v = normal(0, L, B, KV, cap, D, dtype=BF), normal(1, L, B, KV, cap, D, dtype=BF)
    mass, pos = normal(2, L, B, KV, cap).abs(), torch.arange(cap, device=DEV, dtype=torch.int32).expand(L, B, KV, cap).contiguous()
    lens, nxt, out = ints([130] * 8), ints([130] * 8), ints([0] * 8)
    mo, po = torch.zeros_like(mass), torch.zeros_like(pos)
    k0 = k.clone()

    def call():
        ops.cache_evict(k, v, lens, mass, pos, nxt, budget=100, recent=10, mass_out=mo, pos_out=po, lens_out=out)

    call()
    want = (k.clone(), mo.clone(), po.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    k.copy_(k0)
    mo.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(mo, want[1]) and torch.equal(po, want[2])


def test_evict_refuses(ops, mrtdf):
    k = normal(0, 1, 2, 20, 64)
    mass, pos, lens = torch.zeros(1, 2, 20, device=DEV), torch.zeros(1, 2, 20, dtype=torch.int32, device=DEV), ints([20])
    for kw in (dict(budget=0), dict(budget=8, recent=5, sinks=4), dict(budget=8, recent=-1), dict(budget=8, lens_out=lens)):
        with pytest.raises(mrtdf.MrtdfError):
            ops.cache_evict(k, k.clone(), lens, mass, pos, ints([20]), **kw)
    with pytest.raises(mrtdf.MrtdfError):
        ops.cache_evict(k, k.clone(), lens, mass, None, ints([20]), budget=4)


# ---- 4-bit products -------------------------------------------------------------------
def unpack(packed):
    p = packed.cpu().numpy()
    q = np.empty((p.shape[0], p.shape[1] * 2), np.float64)
    q[:, 0::2], q[:, 1::2] = p & 15, p >> 4
    return torch.from_numpy(q)


def q4_case(seed, dtype, m, n, k, group):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    scales = (torch.rand(n, k // group, generator=g) * 0.01 + 0.001).to(dtype).to(DEV)
    biases = (scales.float() * normal(seed + 1, n, k // group).sub(7.5)).to(dtype)
    return normal(seed + 2, m, k, dtype=dtype), packed, scales, biases


def check_q4(ops, x, packed, scales, biases, **kw):
    y = ops.q4_linear(x, packed, scales, biases, **kw)
    k = x.shape[1]
    group = k // scales.shape[1]
    q = unpack(packed)
    s, b = (t.cpu().double().repeat_interleave(group, 1) for t in (scales, biases))
    xd = x.cpu().double()
    want = xd @ (s * q + b).T
    size = xd.abs() @ (s * (q - 8).abs() + (b + 8 * s).abs()).T
    near(y, want, half_step(y.dtype) * want.abs() + size * (group + k // group + 32) * 2.0**-23)
    return y


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16, 17, 33, 64])
def test_q4_rows_and_groups(ops, dtype, group, m):
    check_q4(ops, *q4_case(m, dtype, m, 37, group * 5, group))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (15, 64, 64), (16, 128, 128), (64, 96, 32), (5000, 160, 32), (9601, 1024, 64),
                                       (100, 12288, 32), (33, 8320, 64), (10000, 4224, 128)])
@pytest.mark.parametrize("m", [1, 7])
def test_q4_sizes(ops, dtype, n, k, group, m):
    check_q4(ops, *q4_case(n, dtype, m, n, k, group))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k,group", [(30, 3324, 5504, 64), (64, 300, 2080, 32), (17, 20000, 256, 128), (9, 130, 131072, 128),
                                         (40, 18944, 512, 64), (3, 16500, 8192, 32), (1, 7, 65536, 64)])
def test_q4_streams_weights(ops, dtype, m, n, k, group):
    """Row blocks that two or more CTAs share, several passes over x, groups
    that no wide load fits."""
    check_q4(ops, *q4_case(m, dtype, m, n, k, group))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", [(1, 1024), (2, 4096), (20, 1024)])
def test_q4_scales_at_odd_addresses(ops, dtype, m, k):
    x, packed, scales, biases = q4_case(m, dtype, m, 70, k, 64)
    want = check_q4(ops, x, packed, scales, biases)

    def moved(t):
        return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)

    for s, b in ((moved(scales), biases), (scales, moved(biases)), (moved(scales), moved(biases))):
        assert (s.data_ptr() | b.data_ptr()) % 16
        assert torch.equal(check_q4(ops, x, packed, s, b), want)


@pytest.mark.parametrize("m", [2, 33])
def test_q4_infinite_scales_stay_in_their_rows(ops, m):
    """k is not a multiple of the kernels' steps: what stands for the columns
    past it must not meet the last group's scale."""
    x, packed, scales, biases = q4_case(m, F32, m, 40, 160, 32)
    x, packed = x.abs() + 0.1, packed | 0x11  # no zero times infinity in the formula
    scales[3, -1] = float("inf")
    y, fine = ops.q4_linear(x, packed, scales, biases), ops.q4_linear(x, packed, scales.clamp(max=1.0), biases)
    assert bool((y[:, 3] == float("inf")).all())
    keep = torch.arange(40, device=DEV) != 3
    assert torch.equal(y[:, keep], fine[:, keep])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("m", [3, 20])
def test_q4_rows_that_are_not_finite_touch_no_other(ops, dtype, value, m):
    x, packed, scales, biases = q4_case(m, dtype, m, 40, 256, 64)
    want = ops.q4_linear(x, packed, scales, biases)
    x[1, 70] = value
    y = ops.q4_linear(x, packed, scales, biases)
    keep = torch.arange(m, device=DEV) != 1
    assert torch.equal(y[keep], want[keep]) and not bool(torch.isfinite(y[1]).any())


def test_q4_out_types_views_and_streams(ops):
    x, packed, scales, biases = q4_case(5, BF, 6, 100, 256, 64)
    a = check_q4(ops, x, packed, scales, biases, out_dtype=F32)
    assert a.dtype == F32
    wide = torch.zeros(6, 512, dtype=BF, device=DEV)
    wide[:, 256:] = x
    base = torch.full((6, 130), 3.0, device=DEV)
    b = check_q4(ops, wide[:, 256:], packed, scales, biases, out=base[:, 5:105])
    assert torch.equal(a, b) and bool((base[:, :5] == 3).all()) and bool((base[:, 105:] == 3).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = ops.q4_linear(x, packed, scales, biases, out_dtype=F32)
    torch.cuda.synchronize()
    assert torch.equal(a, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d = ops.q4_linear(x, packed, scales, biases, out_dtype=F32)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, d)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_q4_quantize(ops, dtype, group):
    w = normal(1, 19, group * 3, dtype=dtype)
    w[2, :group] = 0.5  # a group of equal values
    w[3, :group] = 0.0
    packed, scales, biases = ops.q4_quantize(w, group)
    f = w.float().cpu().view(19, 3, group)
    lo, hi = f.amin(2), f.amax(2)
    s, b = ((hi - lo) / 15).to(dtype), lo.to(dtype)
    q = torch.where(s.float()[..., None] > 0, torch.round((f - b.float()[..., None]) / s.float()[..., None]), torch.zeros(())).clamp(0, 15)
    assert torch.equal(scales.cpu(), s) and torch.equal(biases.cpu(), b)
    assert torch.equal(unpack(packed).float(), q.reshape(19, -1))
    # half a step of the code (and of the rounded scale and bias) from w
    err = (s.double()[..., None] * q.double() + b.double()[..., None] - f.double()).abs()
    most = s.double()[..., None] * (0.5 + 15 * half_step(dtype)) + f.abs().double().amax(2, keepdim=True) * 2 * half_step(dtype)
    assert bool((err <= most).all())


def test_q4_refuses(ops, mrtdf):
    x, packed, scales, biases = q4_case(5, F32, 2, 10, 128, 64)
    for f in (lambda: ops.q4_linear(x.half(), packed, scales, biases), lambda: ops.q4_linear(x, packed[:, :32], scales, biases),
              lambda: ops.q4_linear(x, packed, scales.bfloat16(), biases), lambda: ops.q4_linear(x, packed, scales, biases, out_dtype=BF),
              lambda: ops.q4_linear(x, packed, torch.zeros(10, 8, device=DEV), torch.zeros(10, 8, device=DEV)),
              lambda: ops.q4_linear(x.T.contiguous().T, packed, scales, biases),
              lambda: ops.q4_linear(normal(0, 65, 128), packed, scales, biases), lambda: ops.q4_quantize(x, 48),
              lambda: ops.q4_linear(torch.zeros(257, device=DEV)[1:].view(2, 128), packed, scales, biases)):
        with pytest.raises(mrtdf.MrtdfError):
            f()


# ---- together ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_run_of_drafts_over_a_bounded_cache(ops, dtype):
    """Verification steps as a decoder makes them: 4-bit projections of the
    drafted tokens, tree attention per layer, collected weight, commit, and
    eviction when the cache is over its budget; every step against the oracles
    on the same inputs, the state carried by the operators."""
    L, B, H, KV, D, N, P, cap, budget, dm = 2, 2, 4, 2, 64, 6, 3, 40, 24, 128
    rng = np.random.default_rng(3)
    k, v = torch.zeros(L, B, KV, cap, D, dtype=dtype, device=DEV), torch.zeros(L, B, KV, cap, D, dtype=dtype, device=DEV)
    mass, pos = torch.zeros(L, B, KV, cap, device=DEV), torch.zeros(L, B, KV, cap, dtype=torch.int32, device=DEV)
    lens, nxt, bias = ints([0, 0]), ints([0, 0]), normal(1, H, 16)
    width = (H + 2 * KV) * D
    weights = [ops.q4_quantize(normal(20 + l, width, dm, dtype=dtype, std=0.05), 32) for l in range(L)]
    for step in range(14):
        x = normal(100 + step, B * N, dm, dtype=dtype)
        parents = ints([tree_of(rng, N) for _ in range(B)])
        ch = [chains(parents[b].cpu(), N) for b in range(B)]
        path = np.full((B, P), -1)
        for b in range(B):  # a chain of the tree: the path of a random node
            c = ch[b][int(rng.integers(0, N))][:P]
            path[b, : len(c)] = c
        path = ints(path.tolist())
        qs, kns, vns, lses = [], [], [], []
        for l in range(L):
            rows = check_q4(ops, x, *weights[l]).view(B, N, H + 2 * KV, D).transpose(1, 2)
            q, kn, vn = rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:]
            _, lse = check_tree(ops, (q, kn, vn, k[l], v[l]), lens, parents, rel_bias=bias, pos=pos[l], next_pos=nxt)
            qs.append(q), kns.append(kn), vns.append(vn), lses.append(lse)
        q, kn, vn, lse = (torch.stack(t) for t in (qs, kns, vns, lses))
        want, tol = collected(q, lse, kn, k, lens, path, mass, mass, rel_bias=bias, pos=pos, next_pos=nxt)
        ops.cache_mass(q, lse, kn, k, lens, path, mass, rel_bias=bias, pos=pos, next_pos=nxt)
        near(mass, want, tol)
        old = lens.tolist()
        lens, nxt = ops.cache_commit(kn, vn, k, v, lens, path, pos=pos, next_pos=nxt)
        for b in range(B):
            mine = [n for n in path[b].tolist() if n >= 0]
            assert int(lens[b]) == old[b] + len(mine)
            assert torch.equal(k[:, b, :, old[b]:int(lens[b])], kn[:, b, :, mine])
        held = [sorted(pos[l, b, h, : int(lens[b])].tolist()) for l in range(L) for b in range(B) for h in range(KV)]
        lens = ops.cache_evict(k, v, lens, mass, pos, nxt, budget=budget, recent=6, sinks=1)
        assert max(lens.tolist()) <= budget
        i = 0
        for l in range(L):
            for b in range(B):
                for h in range(KV):
                    now = pos[l, b, h, : int(lens[b])].tolist()
                    assert len(set(now)) == len(now) and set(now) <= set(held[i])
                    assert {0} | set(range(max(0, int(nxt[b]) - 6), int(nxt[b]))) <= set(now)
                    i += 1
    assert int(nxt.max()) > budget


@pytest.mark.parametrize("dtype", [0, 1])
def test_stream_cache_is_the_streams_own(ops, mrtdf, tiny_weights, dtype):
    """mrtdf_stream_cache: the caches that the engine's layers attend over, as
    operands. What the engine put there comes back, and a cross-attention step
    over it agrees with the oracle."""
    cfg = mrtdf.preset("tiny", dtype)
    eng = mrtdf.Engine(cfg).load_safetensors(tiny_weights)
    st = mrtdf.Stream(eng, 1, True)
    t = BF if dtype else F32
    rng = np.random.default_rng(5)
    H, S = cfg.num_heads, cfg.max_encoder_length
    hk, hv = (rng.standard_normal((2, H, S, 64)).astype(np.float32) for _ in range(2))
    layer = cfg.num_temporal_layers - 1
    st.probe_set_cache(2, layer, hk, hv)
    k, v, n = ops.stream_cache(st, 2)
    assert n == S and k.shape == (cfg.num_temporal_layers, 2, H, S, 64) and k.dtype == t
    assert torch.equal(k[layer].cpu(), torch.from_numpy(hk).to(t)) and torch.equal(v[layer].cpu(), torch.from_numpy(hv).to(t))
    q, kn, vn = (normal(i, 2, H, 1, 64, dtype=t, std=0.2) for i in range(3))
    check_tree(ops, (q, kn, vn, k[layer], v[layer]), ints([S, S]), None)
    for kind, cap, layers in ((0, cfg.max_frames, cfg.num_temporal_layers), (1, cfg.rvq_depth, cfg.num_depth_layers)):
        assert ops.stream_cache(st, kind)[0].shape == (layers, 2, H, cap, 64)
    with pytest.raises(mrtdf.MrtdfError):
        ops.stream_cache(st, 3)
    st.close()
    eng.close()


# ---- the tcgen05 form of tree attention (bf16, more than 16 rows, long caches) ----------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV,N,cap", [(2, 2, 17, 300), (4, 1, 32, 520), (4, 2, 64, 1000), (8, 1, 64, 700), (3, 1, 43, 2100), (16, 1, 64, 400)])
def test_tree_many_rows(ops, D, H, KV, N, cap):
    """17 to 1024 rows per kv head: one block of 128 rows and several, ragged."""
    rng = np.random.default_rng(N + cap)
    lens = [cap, 0, 1, 64 * (cap // 64), cap - 1, -3]
    parents = ints([tree_of(rng, N, N // 4 if b == 4 else 0) for b in range(6)])
    check_tree(ops, tree_inputs(N, BF, 6, H, KV, N, D, cap), ints(lens), parents)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rel_len,stored", [(64, False), (64, True), (2000, True), (1, False)])
def test_tree_many_rows_with_bias(ops, D, rel_len, stored):
    B, H, KV, N, cap = 3, 8, 2, 12, 900
    rng = np.random.default_rng(rel_len)
    kw = dict(rel_bias=normal(9, H, rel_len))
    if stored:
        pos = torch.stack([torch.from_numpy(rng.permutation(3 * cap)[:cap]) for _ in range(B * KV)])
        kw |= dict(pos=pos.view(B, KV, cap).to(torch.int32).to(DEV), next_pos=ints([3 * cap, 3 * cap + 5, 4 * cap]))
    parents = ints([tree_of(rng, N, 2) for _ in range(B)])
    check_tree(ops, tree_inputs(cap, BF, B, H, KV, N, D, cap), ints([cap, 7, 450]), parents, **kw)


def test_tree_many_rows_values_that_are_not_seen(ops):
    """NaN and infinities behind the length, in absent nodes and in a branch that
    other branches do not see; an infinity that a row does see stays one."""
    B, H, KV, N, cap = 2, 8, 2, 6, 700
    q, kn, vn, k, v = tree_inputs(5, BF, B, H, KV, N, 64, cap)
    lens = ints([cap - 30, 0])
    for b in range(B):
        k[b, :, int(lens[b]):], v[b, :, int(lens[b]):] = math.nan, math.inf
    parents = ints([[-1, 0, -1, 2, -2, 4]] * B)
    kn[:, :, 4:], vn[:, :, 4:], q[:, :, 4:] = math.nan, -math.inf, math.nan
    vn[:, :, 3, 5], vn[:, :, 3, 6] = math.inf, math.nan
    out, lse = ops.tree_attention(q, kn, vn, k, v, lens, parents)
    zero = [t.clone() for t in (q, kn, vn, k, v)]
    for t in zero:
        t[~torch.isfinite(t)] = 0
    wo, wl, to, tl = attend(*zero, lens, parents)
    near(lse, wl, tl)
    assert bool((out[:, :, 3, 5] == math.inf).all()) and bool(torch.isnan(out[:, :, 3, 6]).all())
    out[:, :, 3, 5:7] = wo[:, :, 3, 5:7].to(out)
    near(out, wo, to)


@pytest.mark.parametrize("scale", [0.125, -0.25, 0.0])
def test_tree_many_rows_scales_and_large_scores(ops, scale):
    """Scores that rise along the cache (the maximum is raised often), a negative
    and a zero scale."""
    x = list(tree_inputs(8, BF, 1, 8, 2, 9, 128, 1500, std=0.5))
    x[3] *= torch.linspace(0.1, 12, 1500, device=DEV)[None, None, :, None].to(BF)
    check_tree(ops, x, ints([1500]), None, scale=scale)


def test_tree_many_rows_strided_and_expanded(ops):
    """A cache with the heads inside the rows, and one shared by two sequences
    through an expanded view (no tensor map takes that: the other kernel)."""
    B, H, KV, N, D, cap = 2, 8, 2, 9, 64, 800
    rows = normal(1, B, N, (H + 2 * KV) * D, dtype=BF, std=0.3).view(B, N, H + 2 * KV, D).transpose(1, 2)
    both = normal(2, B, cap, 2, KV, D, dtype=BF)
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    a = check_tree(ops, (rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:], k, v), ints([cap, 77]), None)
    one = (rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:], k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))
    b = check_tree(ops, one, ints([cap, 77]), None)
    assert torch.equal(a[1].isfinite(), b[1].isfinite())


def test_tree_many_rows_same_every_time_and_captured(ops):
    x = tree_inputs(9, BF, 3, 16, 2, 12, 128, 1500)
    lens = ints([1500, 3, 800])
    first = ops.tree_attention(*x, lens)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.tree_attention(*x, lens)
        graphs.append((g, r, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, r, _ in graphs:
        assert torch.equal(first[0], r[0]) and torch.equal(first[1], r[1])
