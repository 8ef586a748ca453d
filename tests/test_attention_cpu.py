"""Refusals and host logic of block selection, block attention and the distance
bias: everything that is checked before any device work."""
from __future__ import annotations

import ctypes
import re

import pytest
import torch
from torch.autograd import forward_ad

import torchbvh_b200 as torchbvh
from torchbvh_b200 import _native
from torchbvh_b200._attention import BlockSelection

VOID = ctypes.c_void_p


def _int64(*values):
    return (ctypes.c_int64 * len(values))(*values)


# ---- Python ---------------------------------------------------------------------------------

def test_exports():
    for name in ("BlockSelection", "select_blocks", "attend_blocks", "distance_bias"):
        assert name in torchbvh.__all__ and hasattr(torchbvh, name)
    assert callable(torchbvh.BVH.select_blocks)


@pytest.mark.parametrize("n", [0, -1, 33, 2.0, "4"])
def test_select_rejects_bad_block_counts(n):
    with pytest.raises(ValueError, match="num_blocks must be 1 to 32"):
        torchbvh.select_blocks(torchbvh.BVHHandle({}), torch.zeros(4, 3), n)


@pytest.mark.parametrize("n", [True, False])
def test_select_rejects_a_truth_value_as_a_block_count(n):
    with pytest.raises(ValueError, match="num_blocks must be 1 to 32"):
        torchbvh.select_blocks(torchbvh.BVHHandle({}), torch.zeros(4, 3), n)


def test_select_rejects_what_is_no_handle():
    with pytest.raises(TypeError, match="must be a BVHHandle returned by build_bvh"):
        torchbvh.select_blocks({}, torch.zeros(4, 3), 4)


def _handle(n=100, dim=3):
    return torchbvh.BVHHandle({"node_aabbs": torch.zeros(4, 2 * dim), "sorted_indices": torch.zeros(n, dtype=torch.int64),
                               "num_leaves": n, "dim": dim})


def _batched(b=2, n=100, dim=3):
    return torchbvh.BatchedBVHHandle({"node_aabbs": torch.zeros(b, 4, 2 * dim), "num_leaves": n, "dim": dim,
                                      "batch_size": b, "sorted_indices": torch.zeros(b, n, dtype=torch.int64)})


def test_select_rejects_bad_queries():
    with pytest.raises(ValueError, match=r"select_blocks: query_points must have shape \(M, D\)"):
        torchbvh.select_blocks(_handle(), torch.zeros(2, 4, 3), 4)
    with pytest.raises(ValueError, match=r"must have shape \(B, M, D\)"):
        torchbvh.select_blocks(_batched(), torch.zeros(4, 3), 4)
    with pytest.raises(ValueError, match="last dimension must match BVH dim"):
        torchbvh.select_blocks(_handle(), torch.zeros(4, 2), 4)
    with pytest.raises(ValueError, match="query_points must be a CUDA tensor"):
        torchbvh.select_blocks(_handle(), torch.zeros(4, 3), 4)
    with pytest.raises(TypeError, match="query_offsets requires a RaggedBVHHandle"):
        torchbvh.select_blocks(_handle(), torch.zeros(4, 3), 4, query_offsets=torch.tensor([0, 4]))
    with pytest.raises(ValueError, match="query_offsets is required"):
        torchbvh.select_blocks(torchbvh.RaggedBVHHandle({}, []), torch.zeros(4, 3), 4)


def test_select_rejects_a_destroyed_handle():
    handle = _handle()
    torchbvh.destroy_bvh(handle)
    with pytest.raises(RuntimeError, match="BVH handle has been destroyed"):
        torchbvh.select_blocks(handle, torch.zeros(4, 3), 4)


class _Streams:
    """The allocator's stream calls, kept: a fake current stream, and what was recorded on which."""

    def __init__(self, monkeypatch):
        self.current, self.capturing, self.recorded = 0, False, []
        monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.recorded.append((t.data_ptr(), s)))
        monkeypatch.setattr(_native, "raw_stream", lambda device: self.current)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.capturing)

        def select(geometry, total, device):
            n = geometry.num_blocks
            return torch.zeros(total, n, dtype=torch.int64), torch.zeros(total, n), torch.zeros(256, dtype=torch.uint8)

        monkeypatch.setattr(_native, "select_blocks", select)
        monkeypatch.setattr(_native.BlockGeometry, "device", property(lambda g: 0, lambda g, v: None))

    def take(self):
        got, self.recorded = set(self.recorded), []
        return got


@pytest.mark.parametrize("built_on", [1, None])
@pytest.mark.parametrize("batched", [False, True])
def test_the_tree_s_memory_is_recorded_on_the_stream_that_selects(monkeypatch, batched, built_on):
    # Its memory goes back to the stream that built it as soon as the caller drops it, while the
    # selection's stream, and later the attention's, may still have to read it.
    streams = _Streams(monkeypatch)
    handle, queries = (_batched(), torch.zeros(2, 5, 3)) if batched else (_handle(), torch.zeros(5, 3))
    handle._fields.update(scene_min=torch.zeros(3), scene_max=torch.ones(3))
    handle._built_on = built_on
    tree = {handle[x].data_ptr() for x in ("node_aabbs", "sorted_indices", "scene_min", "scene_max")}
    streams.current = 2
    selection = torchbvh.select_blocks(handle, queries, 4)
    assert streams.take() == {(p, 2) for p in tree}
    selection._stream = 2  # (a device tensor's)
    selection._used_here()
    assert not streams.take()
    streams.current = 1  # the tree's own stream: the selection's memory is what it reads of others
    selection._used_here()
    assert streams.take() >= {(selection._keep[2].data_ptr(), 1)}
    if built_on is not None:
        torchbvh.select_blocks(handle, queries, 4)
        assert not streams.take()
    streams.current, streams.capturing = 3, True
    torchbvh.select_blocks(handle, queries, 4)
    assert not streams.take()


@pytest.mark.parametrize("fails", [False, True])
@pytest.mark.parametrize("name", ["select_blocks", "sorted", "ragged", "attend_blocks", "attend_blocks_backward",
                                  "distance_bias", "distance_bias_backward"])
def test_the_current_device_stays_the_caller_s(monkeypatch, name, fails):
    # A library whose entries make another device the current one, as they do for tensors there.
    current = [0]

    class Library:
        def __getattr__(self, entry):
            def call(*args):
                current[0] = 1
                return 256 if entry.endswith("_size") else _native.TBVH_ERR_BAD_ARG if fails else 0
            return (lambda: b"refused") if entry == "tbvh_last_error" else call

    monkeypatch.setattr(_native, "load_library", Library)
    monkeypatch.setattr(_native, "raw_stream", lambda device: 0)
    monkeypatch.setattr(_native, "_stream", lambda device: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: current.__setitem__(0, d))
    q, k, v = _qkv()
    table, edges, stats, d2 = torch.zeros(2, 4), torch.zeros(3), torch.zeros(5, 2, 2), torch.zeros(1, 10, 4)
    if name in ("sorted", "ragged"):
        monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        monkeypatch.setattr(_native.BlockGeometry, "device", property(lambda g: 0, lambda g, x: None))
        monkeypatch.setattr(_native, "block_table", lambda *a: (ctypes.c_int64 * 7)())
        monkeypatch.setattr(_native, "select_blocks", lambda g, m, d: (torch.zeros(m, 4), torch.zeros(m, 4), None))
        handle, m, offsets = _handle(), 16385, None
        handle._fields.update(scene_min=torch.zeros(3), scene_max=torch.ones(3))
        if name == "ragged":
            offsets = torch.tensor([0, m])
            handle = torchbvh.RaggedBVHHandle({"batch_size": 1}, [], {**handle._fields, "point_offsets": [0, 100]})
        call = lambda: torchbvh.select_blocks(handle, torch.zeros(m, 3), 4, query_offsets=offsets)
    else:
        call = {
            "select_blocks": lambda: _native.select_blocks(_geometry(), 5, torch.device("cpu")),
            "attend_blocks": lambda: _native.attend_blocks(_geometry(), q, k, v, table, edges, 1.0, True, False),
            "attend_blocks_backward": lambda: _native.attend_blocks_backward(
                _geometry(), q, k, v, table, edges, 1.0, q, None, stats, q, True, True, True),
            "distance_bias": lambda: _native.distance_bias(d2, 2, False, table, edges),
            "distance_bias_backward": lambda: _native.distance_bias_backward(d2, 2, False, edges, torch.zeros(1, 10, 2, 4)),
        }[name]
    if fails:
        with pytest.raises(RuntimeError, match="refused"):
            call()
    else:
        call()
    assert current[0] == 0


def _selection(query_shape=(5,), key_shape=(100,), backward=1):
    fields = {"block_indices": torch.zeros(*query_shape, 4, dtype=torch.int64), "num_blocks": 4}
    return BlockSelection(fields, _native.BlockGeometry(backward=backward), (), key_shape, query_shape)


def _qkv(h=2, kv=2, c=8, dtype=torch.float32, m=5, n=100):
    return torch.zeros(m, h, c, dtype=dtype), torch.zeros(n, kv, c, dtype=dtype), torch.zeros(n, kv, c, dtype=dtype)


def test_attend_rejects_what_is_no_selection():
    with pytest.raises(TypeError, match="must be a BlockSelection"):
        torchbvh.attend_blocks({}, *_qkv())
    gone = _selection()
    torchbvh.destroy_bvh(gone)
    with pytest.raises(RuntimeError, match="Block selection has been destroyed"):
        torchbvh.attend_blocks(gone, *_qkv())


def test_attend_rejects_bad_shapes():
    q, k, v = _qkv()
    attend = lambda *a, **kw: torchbvh.attend_blocks(_selection(), *a, **kw)
    with pytest.raises(ValueError, match=r"queries must have shape \(5, H, C\)"):
        attend(q[:4], k, v)
    with pytest.raises(ValueError, match=r"queries must have shape"):
        attend(q[None], k, v)
    with pytest.raises(ValueError, match=r"keys must have shape \(100, Hkv, C\)"):
        attend(q, k[:99], v)
    with pytest.raises(ValueError, match="values must have shape"):
        attend(q, k, v[..., :4])
    with pytest.raises(ValueError, match="keys and values must have the same heads"):
        attend(q, k, v[:, :1])
    with pytest.raises(ValueError, match="query heads must be a multiple of key heads"):
        attend(*_qkv(h=3, kv=2))
    with pytest.raises(ValueError, match="query heads must be a multiple of key heads"):
        attend(*_qkv(h=0, kv=0))
    for c in (0, 129):
        with pytest.raises(ValueError, match="channels must be 1 to 128"):
            attend(*_qkv(c=c))
    with pytest.raises(ValueError, match="queries must be a CUDA tensor"):
        attend(q, k, v)


@pytest.mark.parametrize("h, kv", [(65, 1), (130, 2), (4097, 4097)])
def test_attend_rejects_too_many_heads(h, kv):
    with pytest.raises(ValueError, match="at most 4096 query heads, and 64 to a key head"):
        torchbvh.attend_blocks(_selection(), *_qkv(h=h, kv=kv, c=1, m=5, n=100))


@pytest.mark.parametrize("scale", [1e39, -1e300, float("nan"), float("-inf")])
def test_attend_rejects_scales_past_float32(scale, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with pytest.raises(ValueError, match="scale must be finite in float32"):
        torchbvh.attend_blocks(_selection(), *_qkv(), scale=scale)


@pytest.mark.parametrize("table, edges, text", [
    (torch.zeros(2, 4), None, "must be given together"),
    (None, torch.zeros(3), "must be given together"),
])
def test_attend_rejects_half_a_bias(table, edges, text, monkeypatch):
    # Past the device checks, which need no device for what is refused after them.
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with pytest.raises(ValueError, match=text):
        torchbvh.attend_blocks(_selection(), *_qkv(), bias_table=table, bias_edges=edges)


def test_attend_rejects_bad_types_biases_and_scales(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    attend = lambda *a, **kw: torchbvh.attend_blocks(_selection(), *a, **kw)
    with pytest.raises(ValueError, match="share one type"):
        attend(*_qkv(dtype=torch.float64))
    q, k, v = _qkv()
    with pytest.raises(ValueError, match="share one type"):
        attend(q, k.half(), v)
    edges = torch.zeros(3)
    for table, match in ((torch.zeros(3, 4), r"bias_table must have shape \(H, num_buckets\)"),
                         (torch.zeros(4), r"bias_table must have shape"),
                         (torch.zeros(2, 0), "1 to 64 buckets"), (torch.zeros(2, 65), "1 to 64 buckets"),
                         (torch.zeros(2, 5), r"bias_edges must have shape \(num_buckets - 1,\)"),
                         (torch.zeros(2, 4).double(), "bias_table must be float32")):
        with pytest.raises(ValueError, match=match):
            attend(q, k, v, bias_table=table, bias_edges=edges)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale must be finite"):
            attend(q, k, v, scale=scale)


def test_attend_refuses_gradients_without_the_backward_lists(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(BlockSelection, "_used_here", lambda self: None)
    q, k, v = _qkv()
    with pytest.raises(ValueError, match="backward=True"):
        torchbvh.attend_blocks(_selection(backward=0), q.requires_grad_(True), k, v)


def test_distance_bias_rejects_bad_arguments(monkeypatch):
    d2, table, edges = torch.zeros(1, 10, 2, 4), torch.zeros(2, 3), torch.zeros(2)
    with pytest.raises(ValueError, match="squared_distances must be a CUDA tensor"):
        torchbvh.distance_bias(d2, table, edges)
    with pytest.raises(ValueError, match="must have shape"):
        torchbvh.distance_bias(d2[0, 0], table, edges)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with pytest.raises(ValueError, match="squared_distances must be float32"):
        torchbvh.distance_bias(d2.half(), table, edges)
    with pytest.raises(ValueError, match="head dimension must match table"):
        torchbvh.distance_bias(d2, torch.zeros(3, 3), edges)
    with pytest.raises(ValueError, match="at least one head"):
        torchbvh.distance_bias(d2[:, :, 0], torch.zeros(0, 3), edges)
    with pytest.raises(ValueError, match="edges must have shape"):
        torchbvh.distance_bias(d2, table, torch.zeros(3))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dual", range(4))
def test_forward_mode_derivatives_are_refused_not_dropped(monkeypatch, dual, grad):
    # A dual tensor need not require a gradient; its tangent must not be lost on the way.
    _Streams(monkeypatch)
    monkeypatch.setattr(_native, "attend_blocks", lambda geometry, q, *rest: (q.clone(), None, None))
    inputs = [*_qkv(), torch.zeros(2, 4)]
    edges = torch.zeros(3)
    with forward_ad.dual_level():
        assert torchbvh.attend_blocks(_selection(), *inputs[:3], bias_table=inputs[3], bias_edges=edges) is not None
        t = inputs[dual].requires_grad_(grad)
        inputs[dual] = forward_ad.make_dual(t, torch.ones_like(t))
        for x in inputs:
            if x is not inputs[dual]:
                x.requires_grad_(grad)
        with pytest.raises(NotImplementedError, match="attend_blocks: forward-mode derivatives"):
            torchbvh.attend_blocks(_selection(), *inputs[:3], bias_table=inputs[3], bias_edges=edges)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="attend_blocks: forward-mode derivatives"):
            torchbvh.attend_blocks(_selection(), *inputs[:3], bias_table=inputs[3], bias_edges=edges)


def test_distance_bias_refuses_forward_mode_derivatives(monkeypatch):
    _Streams(monkeypatch)
    monkeypatch.setattr(_native, "distance_bias", lambda d2, heads, *rest: torch.zeros(1, 10, heads, 4))
    d2, edges = torch.zeros(1, 10, 4), torch.zeros(2)
    with forward_ad.dual_level():
        # Buckets do not change with the distances: their derivative is zero.
        assert torchbvh.distance_bias(forward_ad.make_dual(d2, torch.ones_like(d2)), torch.zeros(2, 3), edges) is not None
        table = forward_ad.make_dual(torch.zeros(2, 3), torch.ones(2, 3))
        with pytest.raises(NotImplementedError, match="distance_bias: forward-mode derivatives"):
            torchbvh.distance_bias(d2, table, edges)


# ---- C ABI ----------------------------------------------------------------------------------

def test_python_s_limits_are_the_library_s():
    from torchbvh_b200 import _attention, _build_lib, _constants

    def value(path, pattern):
        (found,) = re.findall(pattern, path.read_text())
        return int(found)

    header, blocks = _build_lib.INCLUDE / "torchbvh_b200.h", _build_lib.CSRC / "tbvh_blocks.h"
    # Were the first lower in the library, larger clouds would keep the caller's order of queries.
    assert _attention._SMALL == value(header, r"TBVH_SMALL_QUERIES = (\d+)")
    assert _constants.MAX_SELECTED_BLOCKS == value(blocks, r"kMaxSelect = (\d+)")
    assert _constants.MAX_BIAS_BUCKETS == value(blocks, r"kMaxBuckets = (\d+)")
    assert _constants.BLOCK_SIZE == 1 << value(blocks, r"kBlockLevels = (\d+)")


def test_block_table(native_lib):
    table = list(_native.block_table([0, 64, 65, 1000], [0, 10, 10, 75]))
    rows = _native.real_node_count
    assert table == [0, 64, 0, 0, 10, 0, 0,
                     64, 1, rows(64), 10, 0, 1, 1,
                     65, 935, rows(64) + rows(1), 10, 65, 1, 2]


@pytest.mark.parametrize("points, queries, text", [
    ((1, 5), (0, 4), "offsets must start at 0"),
    ((0, 5), (2, 4), "offsets must start at 0"),
    ((0, 5, 5), (0, 1, 2), "strictly increasing"),
    ((0, 5, 6), (0, 2, 1), "must not decrease"),
])
def test_block_table_rejects(native_lib, points, queries, text):
    with pytest.raises(RuntimeError, match=text):
        _native.block_table(list(points), list(queries))
    assert native_lib.tbvh_block_table(0, None, None, None) == _native.TBVH_ERR_BAD_ARG


def _geometry(**kw):
    base = dict(device=-1, dim=3, num_blocks=4, backward=0, num_clouds=2, points_per_cloud=1000, queries_per_cloud=70)
    return _native.BlockGeometry(**{**base, **kw})


def _features(**kw):
    base = dict(dtype=0, heads=4, kv_heads=2, channels=32, scale=1.0, num_buckets=0, queries=16, keys=16, values=16)
    return _native.AttendFeatures(**{**base, **kw})


def test_plan_size(native_lib):
    size = lambda **kw: native_lib.tbvh_block_plan_size(ctypes.byref(_geometry(**kw)))
    tiles, entries = 2 * 3, 16  # 32-query tiles; 16 blocks a cloud are fewer than 32 x 4
    assert size() >= tiles * (32 * 4 + 3 * 32 * 4 + 4 + entries * 8)
    assert size(backward=1) >= size() + 2 * tiles * entries * 8
    assert size(points_per_cloud=2**20, num_clouds=1) > size(points_per_cloud=2**12, num_clouds=1)
    assert size(dim=4) == 0 and size(num_blocks=33) == 0 and size(num_clouds=0) == 0
    # Offsets past 32 bits are counted in 64.
    assert size(points_per_cloud=2**30, queries_per_cloud=2**30, num_clouds=1, num_blocks=32) > 2**36


def test_plan_rejects_more_tiles_than_the_backward_lists_can_number(native_lib):
    # Query slots of the lists are 32 bits: at most 2^27 tiles, of which each small cloud has its own.
    size = lambda **kw: native_lib.tbvh_block_plan_size(
        ctypes.byref(_geometry(points_per_cloud=1, queries_per_cloud=1, **kw)))
    assert size(num_clouds=2**27, backward=1) > 0
    assert size(num_clouds=2**27 + 1) > 0
    assert size(num_clouds=2**27 + 1, backward=1) == 0
    assert "too many clouds" in native_lib.tbvh_last_error().decode()


@pytest.mark.parametrize("change, text", [
    ({"dim": 4}, "D must be 2 or 3"),
    ({"num_blocks": 0}, "num_blocks must be 1 to 32"),
    ({"num_clouds": 0}, "number of clouds"),
    ({"points_per_cloud": 2**31}, "total point count"),
    ({"queries_per_cloud": 2**31 - 1}, "total query count"),
    ({"queries_per_cloud": -1}, "total query count"),
    ({"points_per_cloud": 0}, "ragged clouds need a host table"),
    ({}, "NULL input pointer"),
])
def test_select_entry_rejects(native_lib, change, text):
    rc = native_lib.tbvh_select_blocks(ctypes.byref(_geometry(**change)), 16, 16, None)
    assert rc == _native.TBVH_ERR_BAD_ARG and text in native_lib.tbvh_last_error().decode()


def test_select_entry_rejects_a_small_plan_and_a_foreign_table(native_lib):
    g = _geometry(node_aabbs=16, sorted_indices=16, plan=16, plan_bytes=64)
    assert native_lib.tbvh_select_blocks(ctypes.byref(g), 16, 16, None) == _native.TBVH_ERR_WORKSPACE
    table = _native.block_table([0, 64, 65], [0, 10, 10])
    table[7] = 63  # the second cloud's first point
    g = _geometry(points_per_cloud=0, table_host=ctypes.cast(table, VOID), table_dev=16)
    assert native_lib.tbvh_select_blocks(ctypes.byref(g), 16, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert "not one of tbvh_block_table" in native_lib.tbvh_last_error().decode()
    assert native_lib.tbvh_select_blocks(None, 16, 16, None) == _native.TBVH_ERR_BAD_ARG


@pytest.mark.parametrize("change, text", [
    ({"dtype": 3}, "float32, float16 or bfloat16"),
    ({"heads": 3}, "positive multiple"),
    ({"heads": 0}, "positive multiple"),
    ({"kv_heads": 0}, "positive multiple"),
    ({"heads": 130, "kv_heads": 2}, "at most 64 query heads"),
    ({"channels": 0}, "channels must be 1 to 128"),
    ({"channels": 129}, "channels must be 1 to 128"),
    ({"num_buckets": 65}, "1 to 64 buckets"),
    ({"num_buckets": 4}, "NULL bias pointer"),
    ({"keys": None}, "NULL input pointer"),
])
def test_attend_entries_reject(native_lib, change, text):
    g, f = _geometry(), _features(**change)
    for rc in (native_lib.tbvh_attend_blocks(ctypes.byref(g), ctypes.byref(f), 16, None, None, None, 0, None),
               native_lib.tbvh_attend_blocks_backward(ctypes.byref(g), ctypes.byref(f), 16, None, 16, 16, 16, None, None,
                                                      None, 16, 2**40, None)):
        assert rc == _native.TBVH_ERR_BAD_ARG and text in native_lib.tbvh_last_error().decode()


@pytest.mark.parametrize("change, text", [
    ({"scale": float("nan")}, "scale must be finite"),
    ({"scale": float("inf")}, "scale must be finite"),
    ({"queries": 18}, "not aligned to its type"),
    ({"keys": 18}, "not aligned to its type"),
    ({"values": 17, "dtype": 2}, "not aligned to its type"),
    ({"bias_table": 18, "bias_edges": 16, "num_buckets": 4}, "not aligned to its type"),
])
def test_attend_entries_reject_scales_and_misaligned_features(native_lib, change, text):
    g, f = _geometry(), _features(**change)
    for rc in (native_lib.tbvh_attend_blocks(ctypes.byref(g), ctypes.byref(f), 16, None, None, None, 0, None),
               native_lib.tbvh_attend_blocks_backward(ctypes.byref(g), ctypes.byref(f), 16, None, 16, 16, 16, None, None,
                                                      None, 16, 2**40, None)):
        assert rc == _native.TBVH_ERR_BAD_ARG and text in native_lib.tbvh_last_error().decode()


@pytest.mark.parametrize("out, stats, exact", [(18, 16, None), (16, 20, None), (16, 16, 18)])
def test_attend_entry_rejects_misaligned_outputs(native_lib, out, stats, exact):
    g = _geometry(node_aabbs=16, sorted_indices=16, plan=256, plan_bytes=2**40)
    f = _features(dtype=0 if exact is None else 1)
    rc = native_lib.tbvh_attend_blocks(ctypes.byref(g), ctypes.byref(f), out, stats, exact, 16, 2**40, None)
    assert rc == _native.TBVH_ERR_BAD_ARG and "not aligned to its type" in native_lib.tbvh_last_error().decode()
    g.plan = 264
    rc = native_lib.tbvh_attend_blocks(ctypes.byref(g), ctypes.byref(f), 16, 16, None, 16, 2**40, None)
    assert rc == _native.TBVH_ERR_BAD_ARG and "multiple of 16 bytes" in native_lib.tbvh_last_error().decode()


@pytest.mark.parametrize("at", range(7))
def test_backward_entry_rejects_misaligned_pointers(native_lib, at):
    g = _geometry(node_aabbs=16, sorted_indices=16, plan=256, plan_bytes=2**40, backward=1)
    f = _features(num_buckets=4, bias_table=16, bias_edges=16)
    pointers = [16, 16, 16, 16, 16, 16, 16, 16]  # out, out_exact, stats, grad_out, grad of q, k, v, table
    pointers[at] = 18
    rc = native_lib.tbvh_attend_blocks_backward(ctypes.byref(g), ctypes.byref(f), *pointers, 16, 2**40, None)
    assert rc == _native.TBVH_ERR_BAD_ARG and "not aligned to its type" in native_lib.tbvh_last_error().decode()


def test_backward_entry_rejects(native_lib):
    g = _geometry(node_aabbs=16, sorted_indices=16, plan=256, plan_bytes=2**40)
    call = lambda *a: native_lib.tbvh_attend_blocks_backward(ctypes.byref(g), ctypes.byref(_features()), *a)
    error = lambda: native_lib.tbvh_last_error().decode()
    assert call(16, None, 16, 16, 16, 16, None, None, 16, 2**40, None) == _native.TBVH_ERR_BAD_ARG
    assert "both be given" in error()
    assert call(16, None, 16, 16, 16, 16, 16, None, 16, 2**40, None) == _native.TBVH_ERR_BAD_ARG
    assert "without the backward lists" in error()
    assert call(16, None, 16, 16, 16, None, None, 16, 16, 2**40, None) == _native.TBVH_ERR_BAD_ARG
    assert "needs a bias" in error()
    assert call(None, None, 16, 16, 16, None, None, None, 16, 2**40, None) == _native.TBVH_ERR_BAD_ARG
    assert call(16, None, 16, 16, 16, None, None, None, 16, 64, None) == _native.TBVH_ERR_WORKSPACE


def test_distance_bias_entries_reject(native_lib):
    bias, back = native_lib.tbvh_distance_bias, native_lib.tbvh_distance_bias_backward
    assert bias(-1, 16, 10, 0, 4, 1, 16, 16, 3, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert bias(-1, 16, 10, 2, 4, 1, 16, 16, 65, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert bias(-1, 16, -1, 2, 4, 1, 16, 16, 3, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert bias(-1, None, 10, 2, 4, 1, 16, 16, 3, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert bias(-1, 16, 10, 2, 4, 1, 16, None, 3, 16, None) == _native.TBVH_ERR_BAD_ARG
    assert bias(-1, None, 0, 2, 4, 1, None, None, 3, None, None) == _native.TBVH_OK
    assert back(-1, 16, 10, 2, 4, 1, 16, 3, 16, 16, None, 0, None) == _native.TBVH_ERR_WORKSPACE
    assert back(-1, 16, 10, 2, 4, 1, 16, 3, None, 16, 16, 2**30, None) == _native.TBVH_ERR_BAD_ARG
    assert native_lib.tbvh_distance_bias_backward_workspace_size(10, 2, 4, 0) == 0
