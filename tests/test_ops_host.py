"""Argument checks of the operators on device buffers (include/mrtdf.h,
"operators"): every refusal comes before the first CUDA call, so it is tested
here with addresses that are never used. No GPU needed."""
from __future__ import annotations

import ctypes
import struct

import pytest

torch = pytest.importorskip("torch")

NOT_A_NUMBER = float("nan")

# sizeof-exact layouts of the C structures (native alignment).
_CACHE = struct.Struct("@QQQ4q7iQQQ")
_TREE = struct.Struct("@Q" + "Q4q" * 4 + "QQQQQiiif0Q")
_MASS = struct.Struct("@Q" + "Q4q" * 2 + "QQQQQiiiiff0Q")
_COMMIT = struct.Struct("@Q" + "Q4q" * 2 + "QQQii0Q")
_EVICT = struct.Struct("@QQQQQiii0Q")
_Q4 = struct.Struct("@QQQQQQQQqq7i0Q")
_PACK = struct.Struct("@QQQQQq5i0Q")


@pytest.fixture(scope="module")
def ops(mrtdf):
    import mrtops

    L = mrtops.lib()
    for n in ("tree_attention", "cache_mass", "cache_commit", "cache_evict"):
        getattr(L, "mrtdf_" + n).argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p]
    L.mrtdf_tree_attention_workspace.argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_size_t)]
    L.mrtdf_q4_linear.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    return mrtops


def rows(ptr=256, sl=0, sb=4096, sh=1024, sn=64):
    return (ptr, sl, sb, sh, sn)


class Call:
    """Fields of one call, packed on demand."""

    def __init__(self, ops):
        self.ops = ops
        self.cache = dict(size=_CACHE.size, k=4096, v=8192, sl=65536, sb=32768, sh=8192, st=64, layers=1, batch=2,
                          kv_heads=2, capacity=128, head_dim=64, dtype=1, device=0, lens=256, pos=0, next_pos=0)
        self.tree = dict(size=_TREE.size, q=rows(), k_new=rows(), v_new=rows(), out=rows(ptr=1024), lse=0, parents=0, rel_bias=0,
                         workspace=0, workspace_bytes=0, heads=4, nodes=8, rel_len=0, scale=1.0)
        self.mass = dict(size=_MASS.size, q=rows(), k_new=rows(), lse=256, path=256, rel_bias=0, mass=256, mass_out=256,
                         heads=4, nodes=8, path_len=4, rel_len=0, scale=1.0, decay=1.0)
        self.commit = dict(size=_COMMIT.size, k_new=rows(), v_new=rows(), path=256, lens_out=512, next_pos_out=0, nodes=8,
                           path_len=4)
        self.evict = dict(size=_EVICT.size, mass=256, mass_out=256, pos_out=256, lens_out=512, budget=64, recent=8, sinks=1)
        self.q4 = dict(size=_Q4.size, x=256, packed=256, scales=256, biases=256, out=512, workspace=256, workspace_bytes=1 << 20,
                       x_stride=16384, out_stride=64, m=16,
                       n=64, k=16384, group=32, dtype=1, out_dtype=1, device=0)
        self.pack = dict(size=_PACK.size, w=256, packed=256, scales=256, biases=256, w_stride=128, n=4, k=128, group=32,
                         dtype=1, device=0)

    def bytes(self, what):
        flat = []
        for v in getattr(self, what).values():
            flat += list(v) if isinstance(v, tuple) else [v]
        return {"cache": _CACHE, "tree": _TREE, "mass": _MASS, "commit": _COMMIT, "evict": _EVICT, "q4": _Q4,
                "pack": _PACK}[what].pack(*flat)

    def run(self, what):
        L = self.ops.lib()
        if what == "workspace":
            size = ctypes.c_size_t()
            rc = L.mrtdf_tree_attention_workspace(self.bytes("cache"), self.bytes("tree"), ctypes.byref(size))
            return rc, size.value
        if what in ("q4", "pack"):
            return getattr(L, {"q4": "mrtdf_q4_linear", "pack": "mrtdf_q4_quantize"}[what])(self.bytes(what), None), 0
        name = {"tree": "tree_attention", "mass": "cache_mass", "commit": "cache_commit", "evict": "cache_evict"}[what]
        return getattr(L, "mrtdf_" + name)(self.bytes("cache"), self.bytes(what), None), 0


BAD_CACHE = [("size", 8), ("k", 0), ("k", 264), ("lens", 0), ("layers", 0), ("batch", 0), ("kv_heads", 0), ("capacity", 0),
             ("head_dim", 96), ("head_dim", 32), ("dtype", 2), ("device", -1), ("st", 60), ("sh", -64), ("sb", 4), ("batch", 1025),
             ("capacity", (1 << 24) + 1), ("pos", 256)]


@pytest.mark.parametrize("what", ["tree", "mass", "commit", "evict"])
@pytest.mark.parametrize("field,value", BAD_CACHE)
def test_cache_fields_are_checked(ops, what, field, value):
    c = Call(ops)
    if what == "evict":
        c.cache["pos"] = c.cache["next_pos"] = 256
        if field == "pos":
            field, value = "next_pos", 0
    c.cache[field] = value
    rc, _ = c.run(what)
    assert rc in (1, 7), ops.lib().mrtdf_last_error()
    assert rc == (7 if field in ("batch", "capacity") and value > 1000 else 1)


@pytest.mark.parametrize("what,field,value,code", [
    ("tree", "size", 0, 1), ("tree", "heads", 3, 1), ("tree", "heads", 0, 1), ("tree", "nodes", 0, 1), ("tree", "nodes", 65, 7),
    ("tree", "heads", 256, 7), ("tree", "q", rows(ptr=0), 1), ("tree", "q", rows(ptr=8), 1), ("tree", "q", rows(sn=65), 1),
    ("tree", "k_new", rows(sb=-64), 1), ("tree", "v_new", rows(ptr=0), 1), ("tree", "out", rows(ptr=0), 1),
    ("tree", "scale", NOT_A_NUMBER, 1), ("tree", "rel_bias", 256, 1),
    ("mass", "size", 1, 1), ("mass", "path_len", 0, 1), ("mass", "path_len", 9, 1), ("mass", "lse", 0, 1), ("mass", "path", 0, 1),
    ("mass", "mass", 0, 1), ("mass", "mass_out", 0, 1), ("mass", "decay", NOT_A_NUMBER, 1), ("mass", "heads", 5, 1),
    ("mass", "q", rows(ptr=4), 1), ("mass", "nodes", 65, 7),
    ("commit", "size", 1, 1), ("commit", "nodes", 0, 1), ("commit", "nodes", 65, 7), ("commit", "path_len", 9, 1),
    ("commit", "path", 0, 1), ("commit", "lens_out", 0, 1), ("commit", "lens_out", 256, 1), ("commit", "next_pos_out", 512, 1),
    ("commit", "k_new", rows(ptr=0), 1), ("commit", "v_new", rows(sh=12), 1),
    ("evict", "size", 1, 1), ("evict", "mass", 0, 1), ("evict", "mass_out", 0, 1), ("evict", "pos_out", 0, 1),
    ("evict", "lens_out", 0, 1), ("evict", "lens_out", 256, 1), ("evict", "budget", 0, 1), ("evict", "recent", -1, 1),
    ("evict", "recent", 64, 1), ("evict", "sinks", -1, 1),
    ("q4", "size", 1, 1), ("q4", "x", 0, 1), ("q4", "x", 264, 1), ("q4", "packed", 0, 1), ("q4", "packed", 260, 1),
    ("q4", "workspace", 0, 1), ("q4", "workspace", 264, 1), ("q4", "workspace_bytes", 64, 1), ("q4", "scales", 0, 1), ("q4", "biases", 0, 1), ("q4", "out", 0, 1), ("q4", "x_stride", 129, 1), ("q4", "out_stride", 63, 1),
    ("q4", "m", 0, 1), ("q4", "m", 65, 7), ("q4", "n", 0, 1), ("q4", "k", 0, 1), ("q4", "k", 120, 1), ("q4", "k", 1 << 18, 7),
    ("q4", "group", 16, 1), ("q4", "dtype", 3, 1), ("q4", "dtype", 0, 1), ("q4", "out_dtype", 5, 1), ("q4", "device", -1, 1),
    ("pack", "size", 1, 1), ("pack", "w", 0, 1), ("pack", "group", 0, 1), ("pack", "k", 100, 1), ("pack", "w_stride", 100, 1),
    ("pack", "dtype", 9, 1), ("pack", "n", 0, 1)])
def test_fields_are_checked(ops, what, field, value, code):
    c = Call(ops)
    if what == "evict":
        c.cache["pos"] = c.cache["next_pos"] = 256
    if field == "scale" or field == "decay" or field in getattr(c, what):
        getattr(c, what)[field] = value
    rc, _ = c.run(what)
    assert rc == code, ops.lib().mrtdf_last_error()


def test_null_structures(ops):
    L = ops.lib()
    c = Call(ops)
    assert L.mrtdf_tree_attention(None, c.bytes("tree"), None) == 1
    for f in ("tree_attention", "cache_mass", "cache_commit"):
        assert getattr(L, "mrtdf_" + f)(c.bytes("cache"), None, None) == 1
    c.cache["pos"] = c.cache["next_pos"] = 256
    assert L.mrtdf_cache_evict(c.bytes("cache"), None, None) == 1
    assert L.mrtdf_q4_linear(None, None) == 1 and L.mrtdf_q4_quantize(None, None) == 1
    assert L.mrtdf_tree_attention_workspace(c.bytes("cache"), c.bytes("tree"), None) == 1
    assert L.mrtdf_stream_cache(None, 0, 0, ctypes.create_string_buffer(_CACHE.size), None) == 1


def test_attention_takes_one_layer(ops):
    c = Call(ops)
    c.cache["layers"] = 2
    assert c.run("tree")[0] == 1


def test_workspace_follows_the_capacity(ops):
    """A cache of a few tiles needs none; a long one is split and joined. A call
    without the workspace it needs is refused."""
    c = Call(ops)
    assert c.run("workspace") == (0, 0)
    c.cache |= dict(capacity=4096, sh=4096 * 64, sb=2 * 4096 * 64)
    rc, need = c.run("workspace")
    assert rc == 0 and need > 0
    c.tree |= dict(workspace=256, workspace_bytes=need - 1)
    assert c.run("tree")[0] == 1
    c.tree |= dict(workspace=260, workspace_bytes=need)
    assert c.run("tree")[0] == 1


@pytest.mark.parametrize("field,extent", [("sl", "layers"), ("sb", "batch"), ("sh", "kv_heads"), ("st", "capacity")])
def test_rows_that_are_written_do_not_share_memory(ops, field, extent):
    """An expanded cache can be read (attention, weight), not written."""
    for what in ("commit", "evict"):
        c = Call(ops)
        c.cache |= {field: 0, extent: max(2, c.cache[extent]), "pos": 256, "next_pos": 256}
        c.commit |= dict(k_new=rows(sl=8192), v_new=rows(sl=8192), next_pos_out=512)
        assert c.run(what)[0] == 1 and b"zero stride" in ops.lib().mrtdf_last_error()
    c = Call(ops)
    if field != "sl":
        c.cache[field] = 0
        assert c.run("workspace")[0] == 0
        c.tree["out"] = rows(ptr=1024, **{{"st": "sn"}.get(field, field): 0})
        assert c.run("workspace")[0] == 1


@pytest.mark.parametrize("what,field,value", [("q4", "scales", 257), ("q4", "biases", 257), ("q4", "out", 257), ("pack", "w", 257),
                                              ("pack", "scales", 257), ("pack", "biases", 255)])
def test_elements_are_aligned(ops, what, field, value):
    c = Call(ops)
    getattr(c, what)[field] = value
    assert c.run(what)[0] == 1


def test_outputs_are_other_buffers_than_inputs(ops):
    for what, change in (("tree", dict(out=rows())), ("tree", dict(out=rows(ptr=4096))), ("tree", dict(out=rows(ptr=8192))),
                         ("q4", dict(out=256)), ("commit", dict(k_new=rows(ptr=4096))), ("commit", dict(v_new=rows(ptr=8192)))):
        c = Call(ops)
        getattr(c, what).update(change)
        assert c.run("workspace" if what == "tree" else what)[0] == 1
        assert b"another buffer" in ops.lib().mrtdf_last_error()


def test_strides_of_single_elements_do_not_matter(ops):
    c = Call(ops)
    c.cache |= dict(batch=1, sb=7, sl=3)
    c.tree |= dict(q=rows(sb=5, sl=1), nodes=1, k_new=rows(sn=3, sb=1), v_new=rows(sn=1, sb=9), out=rows(ptr=1024, sn=2, sb=3))
    c.tree["q"] = rows(sb=5, sn=9)
    assert c.run("workspace")[0] == 0


def test_python_refuses_without_a_gpu(ops, mrtdf):
    k = torch.zeros(1, 1, 8, 64)
    with pytest.raises(mrtdf.MrtdfError, match="CUDA"):
        ops.tree_attention(k[:, :, :1], k[:, :, :1], k[:, :, :1], k, k, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(mrtdf.MrtdfError, match="CUDA"):
        ops.q4_linear(torch.zeros(1, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1), torch.zeros(4, 1))
    with pytest.raises(mrtdf.MrtdfError, match="group"):
        ops.q4_quantize(torch.zeros(4, 64), 48)
