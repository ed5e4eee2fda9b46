"""The operators on device buffers (mrtops.py) where values are not finite, very
large, or all of one sign. Oracles and tolerances: test_ops_gpu.py."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_ops_gpu import (  # noqa: E402,F401
    BF, DEV, F32, attend, check_q4, check_tree, collected, half_step, ints, near, normal, ops, q4_case, tree_inputs,
    unpack)

pytestmark = pytest.mark.gpu

# dtype, D, heads, kv heads, nodes: few rows and many (the tcgen05 kernel where
# the cache is long and bf16).
TREES = [(BF, 64, 2, 1, 3), (F32, 64, 2, 1, 3), (F32, 128, 4, 2, 5), (BF, 128, 16, 1, 8), (BF, 64, 16, 1, 8), (F32, 64, 16, 1, 8)]


@pytest.mark.parametrize("dtype,D,H,KV,N", TREES)
@pytest.mark.parametrize("cap", [200, 6000])
def test_tree_nan_query_gives_nan_however_it_is_split(ops, dtype, D, H, KV, N, cap):
    """A row of NaN scores is NaN, in whole items and in those that several CTAs
    share; the rows beside it are untouched."""
    x = tree_inputs(3, dtype, 1, H, KV, N, D, cap)
    lens = ints([cap - 5])
    wo, wl, to, tl = attend(*x, lens)
    x[0][0, 1, 0, 7] = math.nan
    out, lse = ops.tree_attention(*x, lens)
    assert bool(torch.isnan(out[0, 1, 0]).all()) and bool(torch.isnan(lse[0, 1, 0]))
    wo[0, 1, 0], wl[0, 1, 0] = 0.0, 0.0
    out[0, 1, 0], lse[0, 1, 0] = 0.0, 0.0
    near(out, wo, to)
    near(lse, wl, tl)


@pytest.mark.parametrize("dtype,D,H,KV,N", TREES)
@pytest.mark.parametrize("cap,first,last", [(200, 70, 130), (6000, 1500, 4500), (6000, 0, 6000)])
def test_tree_nan_keys_that_rows_see_give_nan(ops, dtype, D, H, KV, N, cap, first, last):
    """Keys that are NaN over more than a CTA's share of the cache."""
    x = tree_inputs(4, dtype, 2, H, KV, N, D, cap)
    x[3][0, :, first:last, 3] = math.nan
    lens = ints([cap, cap])
    wo, wl, to, tl = attend(*(t[1:] for t in x), lens[1:])
    out, lse = ops.tree_attention(*x, lens)
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(lse[0]).all())
    near(out[1:], wo, to)
    near(lse[1:], wl, tl)


@pytest.mark.parametrize("dtype,D,H,KV,N", TREES)
@pytest.mark.parametrize("cap", [200, 6000])
def test_tree_nan_value_of_a_far_smaller_weight(ops, dtype, D, H, KV, N, cap):
    """A NaN value that a row sees with a weight that underflows: 0 x NaN, in the
    same CTA as the large weights or in another."""
    x = tree_inputs(5, dtype, 1, H, KV, N, D, cap)
    x[0][:], x[3][:, :, : cap // 2] = 1.0, -320.0 / D
    lens = ints([cap])
    wo, wl, to, tl = attend(*x, lens)
    x[4][0, :, 7, 3] = math.nan
    out, lse = ops.tree_attention(*x, lens)
    near(lse, wl, tl)
    assert bool(torch.isnan(out[..., 3]).all())
    out[..., 3], wo[..., 3] = 0.0, 0.0
    near(out, wo, to)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bias", [0, 16])
@pytest.mark.parametrize("cap", [60, 300])
def test_mass_rows_that_count_for_nothing(ops, dtype, bias, cap):
    """Rows with lse = -inf add nothing whatever their scores are; nor do the
    rows that fill a product up."""
    L, B, H, KV, N, D = 1, 2, 3, 1, 5, 64
    q, k, kn = normal(1, L, B, H, N, D, dtype=dtype, std=0.2), normal(2, L, B, KV, cap, D, dtype=dtype), normal(3, L, B, KV, N, D, dtype=dtype)
    lse = torch.full((L, B, H, N), -math.inf, device=DEV)
    lse[0, 1] = 3.0  # the second sequence's rows count
    k[0, 0, 0, 7, 3], k[0, 0, 0, 20] = math.nan, math.inf
    kn[0, 0, 0, 1] = math.nan
    mass, path = normal(5, L, B, KV, cap).abs(), ints([[1, 4, -1], [0, 2, 3]])
    lens = ints([cap - 10, cap - 20])
    kw = dict(decay=0.5)
    if bias:
        kw |= dict(rel_bias=normal(7, H, bias))
    got = ops.cache_mass(q, lse, kn, k, lens, path, mass, mass_out=torch.full_like(mass, -7.0), **kw)
    t = cap - 10
    assert torch.equal(got[0, 0, 0, :t], 0.5 * mass[0, 0, 0, :t])
    assert not got[0, 0, 0, t:t + 2].any() and bool((got[0, 0, 0, t + 2:] == -7).all())
    k[0, 0], kn[0, 0] = 0.0, 0.0
    want, tol = collected(q, lse, kn, k, lens, path, mass, torch.full_like(mass, -7.0), **kw)
    near(got[:, 1], want[:, 1], tol[:, 1])


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_mass_of_an_infinite_key_is_its_own_rows(ops, sign):
    """A key with an infinity weighs what the real rows say: exp(-inf) = 0 or
    infinity, not what a row of zeros would make of it."""
    q, k, kn = normal(1, 1, 1, 2, 3, 64, dtype=BF), normal(2, 1, 1, 1, 200, 64, dtype=BF), normal(3, 1, 1, 1, 3, 64, dtype=BF)
    q[..., 9] = 0.5
    k[0, 0, 0, 11, 9] = -sign * math.inf
    mass, lse = torch.ones(1, 1, 1, 200, device=DEV), torch.full((1, 1, 2, 3), 5.0, device=DEV)
    got = ops.cache_mass(q, lse, kn, k, ints([150]), ints([[0, 2]]), mass.clone())
    assert float(got[0, 0, 0, 11]) == (1.0 if sign > 0 else math.inf)
    assert bool(torch.isfinite(got[0, 0, 0, 12:]).all())


@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("m,n,k,group", [(4, 4096, 1024, 64), (8, 4096, 8192, 128), (32, 2048, 8192, 32)])
def test_q4_values_of_one_sign_lean_to_no_side(ops, dtype, out, m, n, k, group):
    """x of one sign, weights of both: what the sums lose may not pile up on one
    side. Rounding the count = m n results moves each by up to u = half a step of
    itself, evenly to both sides, their mean by 6 u / sqrt(3 count) of their root
    mean square at most. In the products of a group with q - 8 up to group / 16
    steps follow one another, each cut off towards zero by 2^-23 of a sum that is
    no larger than |x| |s (q - 8)| over the group; the rest is rounded evenly."""
    x, packed, scales, biases = q4_case(m, dtype, m, n, k, group)
    x = x.abs()
    y = check_q4(ops, x, packed, scales, biases, out_dtype=out)
    s, b = (t.cpu().double().repeat_interleave(group, 1) for t in (scales, biases))
    q, xd = unpack(packed), x.cpu().double()
    want, size = xd @ (s * q + b).T, xd @ (s * (q - 8).abs()).T
    rms = float(want.square().mean().sqrt())
    lean = float((y.cpu().double() - want).mean())
    assert abs(lean) <= 6 * half_step(out) / math.sqrt(3 * m * n) * rms + group / 16 * 2.0**-23 * float(size.mean()) + 2.0**-22 * rms


@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("m", [1, 4, 8, 33])
@pytest.mark.parametrize("value,size", [(1e36, 1), (2e38, 1), (2e37, 128)])
def test_q4_large_finite_values(ops, dtype, out, m, value, size):
    """x near the largest number of its type, one value of a group or all of
    them: results that are finite come out finite."""
    x, packed, scales, biases = q4_case(m, dtype, m, 50, 384, 128)
    x[m // 2, 128:128 + size] = value
    y = check_q4(ops, x, packed, scales, biases, out_dtype=out)
    assert bool(torch.isfinite(y).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k,group", [(64, 1 << 17, 256, 32), (33, 100000, 128, 64), (64, 1 << 17, 512, 32)])
def test_q4_is_done_when_the_next_kernel_starts(ops, dtype, m, n, k, group):
    """The stream goes on when the result is whole, also where no row block is
    shared and nothing is joined (k up to 256)."""
    x, packed, scales, biases = q4_case(m, dtype, m, n, k, group)
    want = ops.q4_linear(x, packed, scales, biases, out_dtype=F32)
    torch.cuda.synchronize()
    out = torch.empty(m, n, device=DEV)
    for _ in range(20):
        out.fill_(math.nan)
        ops.q4_linear(x, packed, scales, biases, out=out)
        assert not int(out.isnan().sum())
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,D,H,KV,N", [(BF, 64, 2, 1, 3), (F32, 64, 2, 1, 3), (BF, 128, 16, 1, 8), (BF, 64, 16, 1, 8)])
@pytest.mark.parametrize("cap", [200, 3000])
def test_tree_infinite_values_that_rows_see_stay_in_their_columns(ops, dtype, D, H, KV, N, cap):
    """Cached infinities and a NaN make their columns not finite, and nothing else."""
    x = tree_inputs(6, dtype, 2, H, KV, N, D, cap)
    lens = ints([cap, cap - 9])
    wo, wl, to, tl = attend(*x, lens)
    x[4][0, :, 5, 3], x[4][0, :, cap - 2, 9], x[4][0, :, 77, D - 1] = math.inf, -math.inf, math.nan
    out, lse = ops.tree_attention(*x, lens)
    near(lse, wl, tl)
    assert not bool(torch.isfinite(out[0][..., [3, 9, D - 1]]).any())
    out[0][..., [3, 9, D - 1]], wo[0][..., [3, 9, D - 1]] = 0.0, 0.0
    near(out, wo, to)


@pytest.mark.parametrize("dtype,D,H,KV,N", TREES)
def test_the_same_calls_repeat_bit_for_bit(ops, dtype, D, H, KV, N):
    """Attention and collected weight over split items; beside other neighbours a
    sequence's results stay within the tolerance."""
    cap, B = 3000, 3
    x = tree_inputs(7, dtype, B, H, KV, N, D, cap)
    lens = ints([cap, 1700, 5])
    out, lse = ops.tree_attention(*x, lens)
    path, mass = ints([list(range(N))] * B), normal(8, B, KV, cap).abs()

    def weight():
        return ops.cache_mass(x[0], lse, x[1], x[3], lens, path, mass, mass_out=torch.zeros_like(mass))

    first = weight()
    for _ in range(5):
        again = ops.tree_attention(*x, lens)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse) and torch.equal(weight(), first)
    wo, wl, to, tl = attend(*(t[:1] for t in x), lens[:1])
    for now in ([cap, 1700, 5], [cap, 0, 64], [cap, cap, cap]):
        out, lse = ops.tree_attention(*x, ints(now))
        near(out[:1], wo, to)
        near(lse[:1], wl, tl)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m", [2, 8, 40])
def test_the_same_products_repeat_bit_for_bit(ops, dtype, m):
    x, packed, scales, biases = q4_case(m, dtype, m, 3333, 2048, 64)
    first = ops.q4_linear(x, packed, scales, biases)
    for _ in range(5):
        assert torch.equal(ops.q4_linear(x, packed, scales, biases), first)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [8, 72, 64])
def test_tree_over_rows_that_share_memory(ops, dtype, D, step):
    """Read-only rows may overlap: a sliding window over one buffer."""
    B, H, KV, N, cap = 1, 16, 2, 8, 1500
    q, kn, vn, _, _ = tree_inputs(1, dtype, B, H, KV, N, D, 8)
    buf = normal(2, cap * step + 4 * D, dtype=dtype)
    k = buf.as_strided((B, KV, cap, D), (0, 16, step, 1))
    v = buf.flip(0).contiguous().as_strided((B, KV, cap, D), (0, 16, step, 1))
    check_tree(ops, (q, kn, vn, k, v), ints([cap - 3]), None)


def test_mass_of_many_rows(ops):
    """1024 query rows of one kv head: sixteen blocks, each onto the sums of the one
    before."""
    L, B, H, KV, N, D, cap = 1, 2, 16, 1, 64, 64, 200
    q, k, kn = normal(1, L, B, H, N, D, dtype=BF, std=0.2), normal(2, L, B, KV, cap, D, dtype=BF), normal(3, L, B, KV, N, D, dtype=BF)
    lse = normal(4, L, B, H, N) + 6
    mass = normal(5, L, B, KV, cap).abs()
    path = ints([list(range(64)), list(range(0, 64))])
    want, tol = collected(q, lse, kn, k, ints([130, 190]), path, mass, torch.zeros_like(mass))
    got = ops.cache_mass(q, lse, kn, k, ints([130, 190]), path, mass, mass_out=torch.zeros_like(mass))
    near(got, want, tol)
