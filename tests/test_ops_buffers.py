"""Operators on device buffers: a buffer that a call writes is no other of its
operands (include/mrtdf.h). Refused before the first CUDA call; no GPU needed."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")

from test_ops_host import Call, ops  # noqa: E402,F401


def apart(ops):
    """A call whose buffers have addresses of their own."""
    c = Call(ops)
    c.cache |= dict(pos=1 << 16, next_pos=2 << 16, lens=3 << 16)
    c.tree |= dict(lse=4 << 16, parents=5 << 16, rel_bias=6 << 16, rel_len=4)
    c.mass |= dict(lse=4 << 16, path=5 << 16, rel_bias=6 << 16, rel_len=4, mass=7 << 16, mass_out=8 << 16)
    c.commit |= dict(path=5 << 16, lens_out=9 << 16, next_pos_out=10 << 16)
    c.evict |= dict(mass=7 << 16, mass_out=8 << 16, pos_out=11 << 16, lens_out=9 << 16)
    return c


NAMES = {1: "pos", 2: "next_pos", 3: "lens", 4: "lse", 5: "parents or path", 6: "rel_bias", 7: "mass", 8: "mass_out", 9: "lens_out",
         11: "pos_out"}


@pytest.mark.parametrize("what,field,at", [
    *[("tree", "lse", i) for i in (1, 2, 3, 5, 6)],
    *[("mass", "mass_out", i) for i in (1, 2, 3, 4, 5, 6)],
    *[("commit", "lens_out", i) for i in (1, 2, 3, 5)], *[("commit", "next_pos_out", i) for i in (1, 2, 3, 5, 9)],
    *[("evict", "lens_out", i) for i in (1, 2, 3, 7, 8, 11)], *[("evict", "pos_out", i) for i in (2, 3, 7, 8)],
    *[("evict", "mass_out", i) for i in (1, 2, 3)]], ids=lambda v: NAMES.get(v, str(v)))
def test_written_buffers_are_no_other_operand(ops, what, field, at):
    c = apart(ops)
    getattr(c, what)[field] = at << 16
    assert c.run("workspace" if what == "tree" else what)[0] == 1
    assert b"another buffer" in ops.lib().mrtdf_last_error()


@pytest.mark.parametrize("where", ["k", "v", "q", "k_new", "v_new", "out"])
def test_lse_is_not_among_the_rows(ops, where):
    c = apart(ops)
    c.tree["lse"] = c.cache[where] if where in "kv" else c.tree[where][0]
    assert c.run("workspace")[0] == 1 and b"another buffer" in ops.lib().mrtdf_last_error()


def test_buffers_of_their_own_are_taken(ops):
    assert apart(ops).run("workspace")[0] == 0
