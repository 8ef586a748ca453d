"""Block selection, block attention and the distance bias on the GPU, against a
float64 oracle (attention_oracle.py)."""
from __future__ import annotations

import ctypes
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

import torchbvh_b200 as torchbvh
from torchbvh_b200 import _native
from tests import attention_oracle as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _cloud(rng, n, dim, kind="uniform"):
    if kind == "same":
        return np.full((n, dim), 0.25, np.float32)
    if kind == "clusters":
        return (rng.random((4, dim))[rng.integers(0, 4, n)] + 0.02 * rng.standard_normal((n, dim))).astype(np.float32)
    return rng.random((n, dim), dtype=np.float32)


class Scene:
    """Clouds in one layout, their queries, and the layout's tensors."""

    def __init__(self, layout, sizes, queries, dim, seed=0, kind="uniform"):
        rng = np.random.default_rng(1000 + seed)
        self.layout, self.sizes, self.queries, self.dim = layout, sizes, queries, dim
        self.points = [_cloud(rng, n, dim, kind) for n in sizes]
        self.qpts = [_cloud(rng, m, dim) for m in queries]
        self.bvh = torchbvh.build_bvh(self.tensor(self.points), batch_offsets=self.offsets(sizes))
        if layout == "ragged":
            self.orders = [h["sorted_indices"].cpu().numpy() for h in self.bvh._require_handles()]
        else:
            self.orders = list(self.bvh["sorted_indices"].view(len(sizes), -1).cpu().numpy())

    def tensor(self, parts):
        parts = [torch.as_tensor(p) for p in parts]
        if self.layout == "single":
            return parts[0].cuda()
        return (torch.stack(parts) if self.layout == "batched" else torch.cat(parts)).cuda()

    def offsets(self, sizes):
        return torch.tensor(np.cumsum([0, *sizes]), device="cuda") if self.layout == "ragged" else None

    def split(self, t, sizes):
        if self.layout == "single":
            return [t]
        return list(t) if self.layout == "batched" else list(torch.split(t, sizes))

    def select(self, n, **kw):
        return torchbvh.select_blocks(self.bvh, self.tensor(self.qpts), n, query_offsets=self.offsets(self.queries), **kw)


SCENES = {
    "one point": ("single", [1], [1], 3),
    "a block less one": ("single", [63], [5], 2),
    "a block": ("single", [64], [33], 3),
    "a block and one": ("single", [65], [32], 2),
    "single 3-D": ("single", [1500], [700], 3),
    "single 2-D": ("single", [4111], [257], 2),
    "deep": ("single", [70001], [97], 3),
    "batch": ("batched", [450] * 3, [129] * 3, 3),
    "batch of tiny queries": ("batched", [301] * 4, [7] * 4, 2),
    "ragged": ("ragged", [64, 1, 700, 129, 2000], [3, 40, 1, 64, 333], 3),
}


@pytest.mark.parametrize("n", [1, 3, 8, 13, 32])
@pytest.mark.parametrize("name", SCENES)
def test_selection_matches_the_definition(name, n):
    scene = Scene(*SCENES[name])
    got = scene.select(n)
    blocks = scene.split(got["block_indices"], scene.queries)
    dist = scene.split(got["squared_distances"], scene.queries)
    for b, order in enumerate(scene.orders):
        want_b, want_d = oracle.select(scene.points[b], order, scene.qpts[b], n)
        assert np.array_equal(blocks[b].cpu().numpy(), want_b)
        assert np.array_equal(dist[b].cpu().numpy().view(np.int32), want_d.view(np.int32))
    assert torchbvh.device_status() == 0


@pytest.mark.parametrize("queries, dim", [
    ([33], 2), ([1024], 3), ([1025], 2), ([4096], 3), ([4097], 2), ([8193], 3), ([12289], 2), ([16384], 3), ([16385], 3),
    ([16384, 2, 5, 40], 3), ([1, 16385, 33], 2),
])
def test_queries_of_every_order_are_all_served(queries, dim):
    scene = Scene("ragged" if len(queries) > 1 else "single", [900] * len(queries), queries, dim, seed=16)
    for q in scene.qpts:  # some beyond the cloud's box, some equal, one not a number
        q[::3] = q[::3] * 4 - 2
        q[1::7] = q[:1]
    scene.qpts[0][len(scene.qpts[0]) // 2, 0] = np.nan
    got = scene.select(3)
    blocks = scene.split(got["block_indices"], scene.queries)
    for b, order in enumerate(scene.orders):
        want, _ = oracle.select(scene.points[b], order, scene.qpts[b], 3)
        assert np.array_equal(blocks[b].cpu().numpy(), want)
    # Every query has one place in the plan: all rows of an attention are written.
    q = scene.tensor([np.zeros((m, 1, 8), np.float32) for m in queries])
    k = scene.tensor([np.ones((900, 1, 8), np.float32)] * len(queries))
    out = torchbvh.attend_blocks(got, q, k, k)
    empty = (got["block_indices"] < 0).all(-1)
    assert int(empty.sum()) == 1
    # A mean of ones: 1 but for the sums' roundings, of at most 192 terms.
    assert bool(((out - (~empty)[..., None, None].float()).abs() <= 192 * 2.0**-23).all())
    assert torchbvh.device_status() == 0


@pytest.mark.parametrize("n", [1, 4, 7, 16, 31])
@pytest.mark.parametrize("points, queries, kind", [
    (1025, 1, "uniform"), (1089, 40, "same"), (20000, 300, "clusters"), (5000, 18943, "uniform"), (5000, 18945, "uniform"),
])
def test_selection_by_several_warps_or_one(points, queries, kind, n):
    # 592 tiles of 32 queries, and clouds of 16 blocks, are where a tile's warps change.
    scene = Scene("single", [points], [queries], 3, seed=17, kind=kind)
    some = scene.qpts[0][::5]
    some[:] = scene.points[0][np.arange(len(some)) % points]  # on the points: many scores of 0
    scene.qpts[0][-1] = np.inf
    got = scene.select(n)
    want_b, want_d = oracle.select(scene.points[0], scene.orders[0], scene.qpts[0], n)
    assert np.array_equal(got["block_indices"].cpu().numpy(), want_b)
    assert np.array_equal(got["squared_distances"].cpu().numpy().view(np.int32), want_d.view(np.int32))
    assert torchbvh.device_status() == 0


@pytest.mark.parametrize("kind", ["same", "clusters"])
def test_selection_ties_go_to_the_lowest_block(kind):
    scene = Scene("single", [5000], [100], 3, kind=kind)
    scene.qpts[0][:50] = scene.points[0][:50]  # inside boxes: many zero distances
    got = scene.select(9)
    want_b, want_d = oracle.select(scene.points[0], scene.orders[0], scene.qpts[0], 9)
    assert np.array_equal(got["block_indices"].cpu().numpy(), want_b)
    assert np.array_equal(got["squared_distances"].cpu().numpy(), want_d)


def test_queries_that_are_not_finite_select_nothing():
    scene = Scene("single", [900], [40], 3)
    scene.qpts[0][3, 1] = np.nan
    scene.qpts[0][7, 0] = np.inf
    scene.qpts[0][9, 2] = -np.inf
    scene.qpts[0][11] = 3e38  # the square overflows
    got = scene.select(4)
    want_b, want_d = oracle.select(scene.points[0], scene.orders[0], scene.qpts[0], 4)
    for row in (3, 7, 9, 11):
        assert (want_b[row] == -1).all()
    assert np.array_equal(got["block_indices"].cpu().numpy(), want_b)
    assert np.array_equal(got["squared_distances"].cpu().numpy(), want_d)
    q = torch.randn((40, 2, 16), device="cuda", requires_grad=True)
    kv = torch.randn((900, 2, 16), device="cuda", requires_grad=True)
    out = torchbvh.attend_blocks(got, q, kv, kv)
    out.sum().backward()
    for row in (3, 7, 9, 11):
        assert not out[row].any() and not q.grad[row].any()
    assert bool(out.isfinite().all()) and bool(q.grad.isfinite().all()) and bool(kv.grad.isfinite().all())


def test_no_queries():
    scene = Scene("batched", [100] * 2, [0] * 2, 3)
    selection = scene.select(4)
    assert selection["block_indices"].shape == (2, 0, 4)
    q = torch.zeros((2, 0, 2, 8), device="cuda", requires_grad=True)
    k = torch.randn((2, 100, 2, 8), device="cuda", requires_grad=True)
    table = torch.zeros((2, 3), device="cuda", requires_grad=True)
    out = torchbvh.attend_blocks(selection, q, k, k, bias_table=table, bias_edges=torch.ones(2, device="cuda"))
    assert out.shape == q.shape
    out.sum().backward()
    assert not k.grad.any() and not table.grad.any() and q.grad.shape == q.shape


def _features(scene, dtype, heads, kv_heads, channels, num_buckets, seed, train=True):
    g = torch.Generator().manual_seed(77 + seed)
    rand = lambda *shape: torch.randn(shape, generator=g)
    make = lambda sizes, h: [rand(n, h, channels).to(dtype) for n in sizes]
    out = {"q": make(scene.queries, heads), "k": make(scene.sizes, kv_heads), "v": make(scene.sizes, kv_heads),
           "grad": make(scene.queries, heads), "table": None, "edges": None}
    if num_buckets:
        out["table"] = rand(heads, num_buckets)
        out["edges"] = torch.logspace(-4, 0.3, num_buckets - 1)
    return out


def _run(scene, selection, f, scale=None, train=True, prepare=lambda t: t):
    """(out, dq, dk, dv, dtable) through the public calls."""
    leaf = lambda t: prepare(t).detach().requires_grad_(train)
    q, k, v = (leaf(scene.tensor(f[x])) for x in "qkv")
    table = None if f["table"] is None else f["table"].cuda().requires_grad_(train)
    edges = None if f["edges"] is None else f["edges"].cuda()
    out = torchbvh.attend_blocks(selection, q, k, v, bias_table=table, bias_edges=edges, scale=scale)
    if not train:
        return (out,)
    leaves = [q, k, v] + ([] if table is None else [table])
    return (out.detach(), *torch.autograd.grad(out, leaves, scene.tensor(f["grad"])))


def _check(scene, selection, f, got, scale=None, train=True):
    chosen = scene.split(selection["block_indices"].cpu(), scene.queries)
    dt = dt_bound = 0
    parts = [scene.split(x.cpu(), s) for x, s in zip(got[:4], (scene.queries, scene.queries, scene.sizes, scene.sizes))]
    for b, order in enumerate(scene.orders):
        want = oracle.Attention(torch.as_tensor(scene.points[b]), order, torch.as_tensor(scene.qpts[b]), chosen[b],
                                f["q"][b], f["k"][b], f["v"][b], f["table"], f["edges"], scale,
                                f["grad"][b] if train else None)
        oracle.within(parts[0][b], want.out, want.out_bound, f"out {b}")
        if train:
            oracle.within(parts[1][b], want.dq, want.dq_bound, f"grad of queries {b}")
            oracle.within(parts[2][b], want.dk, want.dk_bound, f"grad of keys {b}")
            oracle.within(parts[3][b], want.dv, want.dv_bound, f"grad of values {b}")
            if f["table"] is not None:
                dt, dt_bound = dt + want.dt, dt_bound + want.dt_bound
    if train and f["table"] is not None:
        oracle.within(got[4], dt, dt_bound, "grad of table")
    assert torchbvh.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("name", SCENES)
def test_attention_and_gradients_by_layout(name, dtype):
    if name == "deep":
        pytest.skip("selection only: the dense oracle is for small clouds")
    scene = Scene(*SCENES[name], seed=3)
    selection = scene.select(3)
    f = _features(scene, dtype, 2, 2, 16, 7, seed=1)
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("channels", [1, 3, 8, 12, 20, 32, 33, 48, 64, 80, 96, 100, 127, 128])
def test_channels(channels, dtype):
    scene = Scene("single", [333], [90], 3, seed=channels)
    selection = scene.select(4)
    f = _features(scene, dtype, 3, 3, channels, 5, seed=channels)
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("channels", [24, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (5, 5), (9, 9), (8, 2), (6, 3), (4, 1), (7, 1), (12, 2), (20, 2)])
def test_heads_that_share_keys(heads, channels, dtype):
    scene = Scene("batched", [200] * 2, [50] * 2, 2, seed=heads[0])
    selection = scene.select(3)
    f = _features(scene, dtype, *heads, channels, 64, seed=heads[0])
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("heads", [(3, 3), (8, 2), (3, 1)])
def test_long_lists(heads, dtype):
    """Blocks that dozens of tiles list, and tiles of dozens of blocks."""
    scene = Scene("single", [700], [1500], 2, seed=heads[0])
    selection = scene.select(6)
    f = _features(scene, dtype, *heads, 20, 9, seed=heads[0])
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("num_buckets", [0, 1, 2, 33, 64])
@pytest.mark.parametrize("dim", [2, 3])
def test_bias_buckets(num_buckets, dim):
    scene = Scene("single", [500], [70], dim, seed=num_buckets)
    selection = scene.select(6)
    f = _features(scene, F32, 4, 2, 16, num_buckets, seed=dim)
    _check(scene, selection, f, _run(scene, selection, f, scale=0.7), scale=0.7)


def test_bias_edges_on_the_distances_in_any_order_and_equal():
    scene = Scene("single", [300], [40], 3, seed=5)
    selection = scene.select(5)
    f = _features(scene, F32, 2, 2, 16, 12, seed=5)
    d2 = oracle.pair_distances(torch.as_tensor(scene.qpts[0]), torch.as_tensor(scene.points[0]))
    exact = d2[3, 10:16]  # borders that pairs hit exactly
    f["edges"] = torch.cat([exact, exact[:2], torch.tensor([0.0, float("inf"), float("nan")])])[torch.randperm(11)]
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_bias_of_minus_infinity_masks_and_leaves_rows_empty(dtype):
    scene = Scene("single", [400], [60], 3, seed=6)
    selection = scene.select(2)
    f = _features(scene, dtype, 3, 3, 16, 6, seed=6)
    f["edges"] = torch.tensor([1e-3, 1e-2, 2e-2, 5e-2, 1e-1])
    f["table"][0, :3] = -torch.inf       # near points are masked for head 0
    f["table"][1, :] = -torch.inf        # head 1 sees nothing at all
    f["table"][2, 4] = torch.finfo(F32).min  # lowest finite value
    got = _run(scene, selection, f)
    assert not got[0][:, 1].any() and not got[1][:, 1].any() and not got[2][:, 1].any() and not got[3][:, 1].any()
    _check(scene, selection, f, got)


def test_nonfinite_rows_reach_only_those_that_attend_to_them():
    scene = Scene("single", [640], [96], 3, seed=8)
    selection = scene.select(2)
    f = _features(scene, BF16, 2, 2, 32, 4, seed=8)
    clean = _run(scene, selection, f)
    order, chosen = scene.orders[0], selection["block_indices"].cpu().numpy()
    bad_block = int(chosen[0, 0])
    touched = (chosen == bad_block).any(1)
    assert touched.any() and not touched.all()
    rows = order[64 * bad_block: 64 * bad_block + 64]
    f["k"][0][rows[0]], f["v"][0][rows[1]] = torch.nan, torch.inf
    got = _run(scene, selection, f)
    for i in (0, 1):  # outputs and query gradients of the other rows are what they were
        assert torch.equal(got[i][~touched], clean[i][~touched])
        assert not bool(got[i][touched].isfinite().all())
    # The other way: rows of queries that are not finite.
    f = _features(scene, BF16, 2, 2, 32, 4, seed=8)
    bad_query = int(np.flatnonzero(touched)[0])
    f["q"][0][bad_query], f["grad"][0][bad_query] = torch.nan, torch.nan
    got = _run(scene, selection, f)
    other = np.ones(640, bool)
    for block in chosen[bad_query]:
        other[order[64 * block: 64 * block + 64]] = False
    for i in (2, 3):
        assert torch.equal(got[i][other], clean[i][other])


def test_large_logits_stay_finite():
    scene = Scene("single", [300], [33], 3, seed=9)
    selection = scene.select(5)
    f = _features(scene, F32, 2, 2, 16, 0, seed=9)
    f["q"][0] *= 300
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 30.0])
def test_half_gradients_keep_their_precision_at_any_size(scale):
    scene = Scene("single", [300], [64], 3, seed=10)
    selection = scene.select(4)
    f = _features(scene, F16, 2, 2, 32, 5, seed=10)
    f["grad"][0] = (f["grad"][0].float() * scale).to(F16)
    got = _run(scene, selection, f)
    _check(scene, selection, f, got)


def test_half_gradients_of_large_values_stay_in_range():
    # <grad, value> is up to 2^17 for a gradient of 1: float16's range has room for it only
    # if the power of two that lifts the gradients looks at the values too.
    scene = Scene("single", [300], [64], 3, seed=13)
    selection = scene.select(4)
    f = _features(scene, F16, 2, 2, 128, 5, seed=13)
    f["v"][0] = (f["v"][0].float() * 4096).clamp(-65000, 65000).to(F16)
    f["grad"][0] = (f["grad"][0].float() * 2.0**-12).to(F16)
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("grad", [2.0**-14, 1.0, 2.0**8])
def test_half_gradients_beside_an_outlying_value(grad):
    # A value that no query sees leaves room for the gradients of the others: 2 * 32 * 4 * 2^10
    # of it are lifted to 2^15, a typical dS of 6 / 256 then to 2^-9, four powers of two above
    # float16's subnormal numbers, whose half step is 2^-4.5 of the rounding that is counted.
    scene = Scene("single", [2000], [64], 3, seed=18)
    scene.qpts[0] *= 0.1
    selection = scene.select(4)
    f = _features(scene, F16, 2, 2, 32, 5, seed=18)
    seen = set(selection["block_indices"].unique().tolist())
    hidden = next(j for j in range(31) if j not in seen)
    f["v"][0][scene.orders[0][64 * hidden]] = 1024.0
    f["grad"][0] = (f["grad"][0].float() * grad).to(F16)
    _check(scene, selection, f, _run(scene, selection, f))


@pytest.mark.parametrize("num_buckets", [0, 3])  # 3: with the output kept in float32
@pytest.mark.parametrize("points, queries, n", [(64, 64, 1), (640, 40, 10)])  # 10: tiles are split
def test_half_weights_far_below_the_largest_keep_their_bits(points, queries, n, num_buckets):
    # One point takes nearly all of every row's weight and has no value: what is left are sums of
    # weights of about 2^-26, which float16 could not hold as they are, times values of 2^8.
    scene = Scene("single", [points], [queries], 3, seed=25)
    selection = scene.select(n)
    f = _features(scene, F16, 2, 2, 32, num_buckets, seed=25)
    q, k, v, grad = (f[x][0] for x in ("q", "k", "v", "grad"))
    q *= 0.25
    q[..., 0], k[..., 0] = 8, 0
    k[5, :, 0] = 12.75  # 8 * 12.75 / 32^0.5 = 18.03
    v *= 256
    v[5] = 0
    grad *= 256
    if num_buckets:
        f["table"].zero_()
    got = _run(scene, selection, f)
    chosen = selection["block_indices"].cpu()
    want = oracle.Attention(torch.as_tensor(scene.points[0]), scene.orders[0], torch.as_tensor(scene.qpts[0]), chosen, q, k, v,
                            f["table"], f["edges"], None, grad)
    others = want.p[:, :, torch.arange(points) != 5]
    assert 2.0**-29 < float(others.min()) and float(others.max()) < 2.0**-22
    # dS is lifted to float16's range by the largest that it could be; below 2^-14 of that range it has
    # half a step of 2^-24 instead of a relative one.
    most = 2 * 32 * float(grad.abs().max()) * float(v.abs().max())
    step = 2.0**-25 / 2.0 ** (14 - np.floor(np.log2(most))) * 32**-0.5
    oracle.within(got[0], want.out, want.out_bound, "out")
    oracle.within(got[1], want.dq, want.dq_bound + step * k.double().abs().sum(0), "grad of queries")
    oracle.within(got[2], want.dk, want.dk_bound + step * q.double().abs().sum(0), "grad of keys")
    oracle.within(got[3], want.dv, want.dv_bound, "grad of values")
    if num_buckets:
        oracle.within(got[4], want.dt, want.dt_bound, "grad of table")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_infinite_values_are_infinite_results(dtype):
    scene = Scene("single", [300], [70], 3, seed=26)
    selection = scene.select(5)  # all blocks
    f = _features(scene, dtype, 2, 2, 40, 0, seed=26)
    clean = _run(scene, selection, f, train=False)[0]
    f["v"][0][7, :, 3], f["v"][0][9, :, 30], f["v"][0][8, :, 12] = torch.inf, -torch.inf, torch.nan
    got = _run(scene, selection, f, train=False)[0]
    assert bool((got[..., 3] == torch.inf).all()) and bool((got[..., 30] == -torch.inf).all())
    assert bool(got[..., 12].isnan().all())
    rest = [c for c in range(40) if c not in (3, 12, 30)]
    assert torch.equal(got[..., rest], clean[..., rest])


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_a_key_that_makes_a_logit_minus_infinity_is_masked(dtype, sign):
    # As one whose logit is so low that its weight is zero: the same bits.
    scene = Scene("single", [300], [70], 3, seed=27)
    selection = scene.select(5)
    f = _features(scene, dtype, 2, 2, 40, 4, seed=27)
    f["q"][0][..., 2] = sign * (f["q"][0][..., 2].abs() + 0.5)
    runs = []
    for low in (-torch.inf, -3e4):
        f["k"][0][11, :, 2] = sign * low
        runs.append(_run(scene, selection, f))
    for i in (0, 3, 4):  # output, gradients of values and table (0 times the key itself is not a number)
        assert bool(runs[0][i].isfinite().all()) and torch.equal(runs[0][i], runs[1][i])
    assert not runs[0][3][11].any()


def test_float32_values_up_to_the_type_s_largest():
    scene = Scene("single", [100], [40], 3, seed=28)
    selection = scene.select(2)
    f = _features(scene, F32, 1, 1, 16, 0, seed=28)
    most = torch.finfo(F32).max
    for row, x in enumerate((most, -most, most * (1 - 2.0**-12), most * (1 - 2.0**-11), most / 2)):
        f["v"][0][row, 0, row] = x
    got = _run(scene, selection, f, train=False)
    _check(scene, selection, f, got, train=False)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("points, queries, n", [(2048, 3, 32), (2048, 400, 32), (64, 5, 1)])
def test_means_of_the_type_s_largest_values(points, queries, n, dtype, train):
    # All weights are equal: the mean of equal values is the value, though their sum is far above
    # the type's largest. Half of the largest, which leaves room for the result's own roundings.
    scene = Scene("single", [points], [queries], 3, seed=31)
    selection = scene.select(n)
    f = _features(scene, dtype, 2, 2, 16, 3, seed=31)
    f["q"][0].zero_()
    f["table"].zero_()
    most = torch.finfo(dtype).max / 2
    f["v"][0][..., 0], f["v"][0][..., 1] = most, -most
    f["grad"][0][..., :2] = 0
    out = _run(scene, selection, f, train=train)[0]
    # Sums of up to 2,048 equal terms, each rounded once as it is added, and the type's rounding.
    bound = (2100 * 2.0**-23 + oracle.HALF_STEP[dtype]) * most
    for c, x in ((0, most), (1, -most)):
        assert bool(((out[..., c].double() - x).abs() <= bound).all()), c


def test_half_gradients_without_queries():
    scene = Scene("single", [100], [0], 3, seed=13)
    selection = scene.select(4)
    for _ in range(2):  # the workspace is not cleared: fill the memory that it may get
        torch.full((1 << 20,), 3e4, device="cuda")
        k = torch.randn((100, 2, 8), device="cuda").half().requires_grad_()
        torchbvh.attend_blocks(selection, torch.zeros((0, 2, 8), device="cuda").half(), k, k).sum().backward()
        assert not k.grad.any()  # (NaN is not zero)


@pytest.mark.parametrize("scale", [None, 1.0, 40.0, 0.0])
@pytest.mark.parametrize("size", [-1e9, 3e7, -1e30, torch.finfo(F32).min, torch.finfo(F32).max])
@pytest.mark.parametrize("queries", [2, 200])
def test_a_bias_that_all_points_share_changes_nothing(queries, size, scale):
    # Without products the logits are the bias alone: their differences are 0 exactly, whatever
    # its size, so every bit of the result is that of no bias.
    scene = Scene("single", [500], [queries], 3, seed=14)
    selection = scene.select(5)
    f = _features(scene, BF16, 2, 2, 32, 3, seed=14)
    f["q"][0].zero_()
    f["table"].zero_()
    want = _run(scene, selection, f, scale=scale)
    f["table"].fill_(size)
    for got, plain in zip(_run(scene, selection, f, scale=scale), want):
        assert torch.equal(got, plain)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_a_row_of_the_lowest_bias_is_the_mean(dtype):
    # What is added to the type's lowest value is rounded away: such logits are equal.
    scene = Scene("batched", [130] * 2, [40] * 2, 2, seed=15)
    selection = scene.select(2)
    f = _features(scene, dtype, 2, 2, 16, 4, seed=15)
    f["table"].fill_(torch.finfo(F32).min)
    got = _run(scene, selection, f)
    assert all(bool(x.isfinite().all()) for x in got)
    f["q"] = [torch.zeros_like(x) for x in f["q"]]
    f["table"].zero_()
    want = _run(scene, selection, f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("queries", [1, 2, 31])
@pytest.mark.parametrize("n", [1, 7, 32])
def test_few_queries_over_many_blocks(queries, n, dtype):
    scene = Scene("single", [2500], [queries], 3, seed=queries)
    selection = scene.select(n, backward=False)
    f = _features(scene, dtype, 4, 2, 64, 32, seed=n)
    _check(scene, selection, f, _run(scene, selection, f, train=False), train=False)
    trained = scene.select(n)
    _check(scene, trained, f, _run(scene, trained, f))


def test_results_do_not_depend_on_the_rest_of_the_batch():
    """A cloud alone and in a batch: equal bits (the tiles are the cloud's own)."""
    scene = Scene("batched", [500] * 3, [300] * 3, 3, seed=11)
    f = _features(scene, BF16, 4, 4, 32, 9, seed=11)
    got = _run(scene, scene.select(4), f)
    one = Scene("single", [500], [300], 3, seed=11)
    one.points, one.qpts = [scene.points[1]], [scene.qpts[1]]
    one.bvh = torchbvh.build_bvh(one.tensor(one.points))
    g = {x: [f[x][1]] if x in ("q", "k", "v", "grad") else f[x] for x in f}
    alone = _run(one, one.select(4), g)
    for i in range(4):
        assert torch.equal(got[i][1], alone[i])


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_equal_inputs_give_equal_bits(dtype):
    scene = Scene("ragged", [3000, 900], [2000, 1500], 3, seed=12, kind="clusters")
    f = _features(scene, dtype, 4, 4, 32, 16, seed=12)
    first = _run(scene, scene.select(8), f)
    for _ in range(3):
        again = _run(scene, scene.select(8), f)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("queries", [3, 500])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_training_and_inference_give_the_same_bits(dtype, queries):
    scene = Scene("single", [2000], [queries], 3, seed=23)
    f = _features(scene, dtype, 4, 2, 32, 16, seed=23)
    trained, plain = scene.select(8), scene.select(8, backward=False)
    assert torch.equal(_run(scene, trained, f)[0], _run(scene, plain, f, train=False)[0])


def test_many_tiles_on_one_block():
    """One block that every tile lists: the long path of the backward lists."""
    scene = Scene("single", [60], [40000], 2, seed=13)
    selection = scene.select(2)
    f = _features(scene, F32, 1, 1, 8, 3, seed=13)
    got = _run(scene, selection, f)
    # One block: every query sees every point.
    q, k, v, do = (f[x][0].double() for x in ("q", "k", "v", "grad"))
    d2 = oracle.pair_distances(torch.as_tensor(scene.qpts[0]), torch.as_tensor(scene.points[0]))
    z = q[:, 0] @ k[:, 0].T * 8**-0.5 + f["table"].double()[0][oracle.buckets(d2, f["edges"])]
    p = torch.softmax(z, -1)
    dv = p.T @ do[:, 0]
    # Sums of 40,000 float32 terms, 1,250 tiles added in turn: (1,250 + 32) half steps of the partial sums
    # (at most the sum of the terms' sizes), and 2^-18 relative for each term.
    bound = (1282 * 2.0**-24 + 2.0**-18) * (p.T @ do[:, 0].abs())
    oracle.within(got[3][:, 0], dv, bound, "grad of values")
    again = _run(scene, scene.select(2), f)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("points, n", [(60, 1), (130, 2)])
def test_lists_of_more_tiles_than_one_window(points, n):
    """More than 2,048 tiles on a block: the long path of the backward lists takes them in windows."""
    queries = 70001
    scene = Scene("single", [points], [queries], 2, seed=29)
    selection = scene.select(n)
    f = _features(scene, F32, 1, 1, 8, 0, seed=29)
    got = _run(scene, selection, f)
    chosen = selection["block_indices"].cpu()
    counts = torch.bincount(chosen.reshape(-1))
    assert int(counts.max()) > 66000  # (so that some block's entries lie in two windows)
    want = oracle.Attention(torch.as_tensor(scene.points[0]), scene.orders[0], torch.as_tensor(scene.qpts[0]), chosen,
                            f["q"][0], f["k"][0], f["v"][0], None, None, None, f["grad"][0])
    oracle.within(got[0], want.out, want.out_bound, "out")
    oracle.within(got[1], want.dq, want.dq_bound, "grad of queries")
    # Sums over queries: a step of 32 is summed by itself and added to at most 2,188 others, each a half
    # step of partial sums that are at most the sum of the terms' sizes; 2^-18 relative for each term of dV.
    p, do = want.p[0], f["grad"][0][:, 0].double()
    bound = (2220 * 2.0**-24 + 2.0**-18) * (p.T @ do.abs())
    oracle.within(got[3][:, 0], want.dv[:, 0], bound, "grad of values")
    oracle.within(got[2], want.dk, want.dk_bound, "grad of keys")
    again = _run(scene, scene.select(n), f)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_a_cloud_alone_and_in_a_batch_that_is_split_otherwise(dtype):
    """How often tiles are split goes by the whole call's tiles: results then differ by roundings,
    each within its bound."""
    scene = Scene("batched", [500] * 3, [2500] * 3, 3, seed=30)
    f = _features(scene, dtype, 4, 4, 32, 9, seed=30)
    one = Scene("single", [500], [2500], 3, seed=30)
    one.points, one.qpts = [scene.points[1]], [scene.qpts[1]]
    one.bvh = torchbvh.build_bvh(one.tensor(one.points))
    g = {x: [f[x][1]] if x in ("q", "k", "v", "grad") else f[x] for x in f}
    for s, features, tiles in ((scene, f, 3 * 79), (one, g, 79)):
        selection = s.select(8)
        _check(s, selection, features, _run(s, selection, features))


FIRST_CALLS = """
import torch, torchbvh_b200 as t
heads, kv, types, buckets, train = {}
selection = t.select_blocks(t.build_bvh(torch.rand(90, 3, device="cuda")), torch.rand(40, 3, device="cuda"), 2)
table, edges = torch.zeros(heads, buckets, device="cuda"), torch.zeros(buckets - 1, device="cuda")
for dtype, channels in types:
    q = torch.randn(40, heads, channels, device="cuda").to(dtype)
    k = torch.randn(90, kv, channels, device="cuda").to(dtype).requires_grad_(train)
    out = t.attend_blocks(selection, q, k, k, bias_table=table, bias_edges=edges)
    if train:
        out.sum().backward()
torch.cuda.synchronize()
"""


@pytest.mark.parametrize("call", [
    # Shared memory of the forward pass: 49,040 bytes beside 256 static ones, where 49,152 are the default.
    (4, 1, [(F32, 20), (F16, 40), (BF16, 64)], 8, False),
    (5, 1, [(F32, 32), (F16, 64), (BF16, 33)], 1, False),
    # The same of the gradients of keys: 48,912 bytes.
    (46, 1, [(F16, 32), (BF16, 8)], 8, True),
])
def test_the_first_call_of_a_process(call):
    """A kernel's limit of shared memory is raised for the process: what an earlier call of other
    shapes may have raised is not there yet."""
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(call)], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("op", ["attend", "bias"])
def test_two_threads_at_once(op):
    """Entries whose kernel is the same but needs different amounts of shared memory, each in a loop
    of its own thread and stream: no launch may find the limit that the other one needs."""
    lib = _native.load_library()
    scene = Scene("single", [65], [3], 3, seed=32)
    selection = scene.select(1)
    calls, results = [], []
    for heads, buckets in ((4, 64), (2, 42)):
        table, edges = torch.randn((heads, buckets), device="cuda"), torch.logspace(-4, 0, buckets - 1, device="cuda")
        if op == "attend":
            f = _features(scene, F32, heads, heads, 32, 0, seed=32)
            q, k, v = (scene.tensor(f[x]) for x in "qkv")
            out, keep = torch.empty_like(q), (q, k, v, table, edges)
            features = _native._attend_features(*keep, 0.2)
            want = torchbvh.attend_blocks(selection, q, k, v, bias_table=table, bias_edges=edges, scale=0.2)
            size = lib.tbvh_attend_blocks_workspace_size(ctypes.byref(selection._geometry), ctypes.byref(features))
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            args = (ctypes.byref(selection._geometry), ctypes.byref(features), out.data_ptr(), None, None, ws.data_ptr(), size)
            calls.append((lib.tbvh_attend_blocks, args, keep, ws))
        else:
            d2, grad = torch.rand((1, 5, 8), device="cuda"), torch.randn((1, 5, heads, 8), device="cuda")
            out = torch.empty_like(table)
            want, = torch.autograd.grad(torchbvh.distance_bias(d2, table.requires_grad_(), edges), table, grad)
            size = lib.tbvh_distance_bias_backward_workspace_size(5, heads, 8, buckets)
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            args = (0, d2.data_ptr(), 5, heads, 8, 0, edges.data_ptr(), buckets, grad.data_ptr(), out.data_ptr(),
                    ws.data_ptr(), size)
            calls.append((lib.tbvh_distance_bias_backward, args, (d2, grad, edges), ws))
        results.append((out, want))
    torch.cuda.synchronize()
    start, codes = threading.Barrier(len(calls)), []

    def repeat(entry, args, *keep):
        stream = torch.cuda.Stream()
        start.wait(30)
        codes.append({entry(*args, stream.cuda_stream) for _ in range(20000)})
        stream.synchronize()

    threads = [threading.Thread(target=repeat, args=call) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert codes == [{0}, {0}]
    assert all(torch.equal(out, want) for out, want in results)


def test_strides_orders_and_alignment():
    scene = Scene("single", [333], [90], 3, seed=14)
    selection = scene.select(4)
    f = _features(scene, BF16, 4, 4, 24, 5, seed=14)
    want = _run(scene, selection, f)

    def turned(t):  # heads and rows swapped in memory
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def offset(t):  # starts 2 bytes into its memory
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        return flat.copy_(t.reshape(-1)).view(t.shape)

    for prepare in (turned, offset):
        got = _run(scene, selection, f, prepare=prepare)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_broadcast_inputs_and_gradients():
    scene = Scene("single", [200], [64], 3, seed=15)
    selection = scene.select(3)
    one = torch.randn((1, 1, 16), device="cuda", requires_grad=True)
    keys = torch.randn((200, 2, 16), device="cuda", requires_grad=True)
    out = torchbvh.attend_blocks(selection, one.expand(64, 2, 16), keys, keys)
    out.sum().backward()  # the incoming gradient is an expanded scalar
    q = one.detach().repeat(64, 2, 1).requires_grad_(True)
    k, v = keys.detach().clone().requires_grad_(True), keys.detach().clone().requires_grad_(True)
    torchbvh.attend_blocks(selection, q, k, v).backward(torch.ones((64, 2, 16), device="cuda"))
    torch.testing.assert_close(one.grad, q.grad.sum((0, 1), keepdim=True), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(keys.grad, k.grad + v.grad, rtol=1e-6, atol=1e-6)


def test_only_the_needed_gradients():
    scene = Scene("single", [200], [64], 3, seed=16)
    selection = scene.select(3)
    f = _features(scene, F32, 2, 2, 16, 5, seed=16)
    want = _run(scene, selection, f)
    for needed in range(4):
        leaves = [scene.tensor(f[x]) for x in "qkv"] + [f["table"].cuda()]
        leaves[needed].requires_grad_(True)
        out = torchbvh.attend_blocks(selection, *leaves[:3], bias_table=leaves[3], bias_edges=f["edges"].cuda())
        out.backward(scene.tensor(f["grad"]))
        assert torch.equal(leaves[needed].grad, want[needed + 1])
        assert all(leaf.grad is None for i, leaf in enumerate(leaves) if i != needed)


def test_gradients_against_differences():
    """Central differences of the kernel's own outputs along random directions, float32.
    With steps of 2^-6 the truncation is of third order (6e-5 of the third derivative, which is of
    the order of the first here) and the rounding noise 2^-21 / 2^-6: both far below 1 %."""
    scene = Scene("single", [300], [80], 3, seed=17)
    selection = scene.select(4)
    f = _features(scene, F32, 2, 1, 16, 6, seed=17)
    got = _run(scene, selection, f)
    weight = scene.tensor(f["grad"]).double()
    g = torch.Generator().manual_seed(5)
    for name, grad in zip(("q", "k", "v", "table"), got[1:]):
        base = f[name] if name == "table" else f[name][0]
        direction = torch.randn(base.shape, generator=g)
        direction /= direction.norm() / base.norm()

        def loss(sign):
            moved = dict(f)
            moved[name] = base + sign * 2.0**-6 * direction
            if name != "table":
                moved[name] = [moved[name]]
            return float((_run(scene, selection, moved, train=False)[0].double() * weight).sum())

        slope = (loss(1) - loss(-1)) / 2.0**-5
        want = float((grad.double().cpu() * direction.double()).sum())
        size = float(grad.double().norm().cpu() * direction.double().norm())
        assert abs(slope - want) <= 0.01 * size, (name, slope, want)


def test_selection_serves_many_layers_and_survives_its_sources():
    scene = Scene("single", [400], [100], 3, seed=18)
    qpts = scene.tensor(scene.qpts)
    selection = torchbvh.select_blocks(scene.bvh, qpts, 4)
    f = _features(scene, F32, 2, 2, 16, 5, seed=18)
    want = _run(scene, selection, f)
    qpts.fill_(float("nan"))  # the selection holds its own copy
    torchbvh.destroy_bvh(scene.bvh)
    got = _run(scene, selection, f)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    _run(scene, selection, _features(scene, BF16, 8, 8, 64, 0, seed=19))
    # A graph that is alive when the selection is destroyed can still be run backward.
    q, k = scene.tensor(f["q"]).requires_grad_(True), scene.tensor(f["k"])
    out = torchbvh.attend_blocks(selection, q, k, k)
    torchbvh.destroy_bvh(selection)
    out.sum().backward()
    assert q.grad is not None
    with pytest.raises(RuntimeError, match="Block selection has been destroyed"):
        torchbvh.attend_blocks(selection, q, k, k)
    with pytest.raises(RuntimeError, match="destroyed"):
        selection["block_indices"]


def test_on_another_stream():
    scene = Scene("single", [3000], [1000], 3, seed=20)
    f = _features(scene, BF16, 4, 4, 32, 8, seed=20)
    want = _run(scene, scene.select(6), f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(scene, scene.select(6), f)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("queries", [200, 20000])  # put in order by the call, and by the sort that reads the tree's box
@pytest.mark.parametrize("layout", ["single", "ragged"])
def test_a_tree_of_another_stream_may_be_dropped_while_it_is_read(layout, queries):
    scene = Scene(layout, [3000], [queries], 3, seed=24)
    points, qpts, offsets, query_offsets = (scene.tensor(scene.points), scene.tensor(scene.qpts), scene.offsets([3000]),
                                            scene.offsets([queries]))
    f = _features(scene, F32, 2, 2, 16, 0, seed=24)
    q, k, v = (scene.tensor(f[x]) for x in "qkv")
    first = torchbvh.select_blocks(scene.bvh, qpts, 4, query_offsets=query_offsets)
    want = first["block_indices"], torchbvh.attend_blocks(first, q, k, v)
    builder, reader = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(builder):
        tree = torchbvh.build_bvh(points, batch_offsets=offsets)
        sizes = [t.numel() * t.element_size() for t in (scene.bvh._packed if layout == "ragged" else scene.bvh).values()
                 if isinstance(t, torch.Tensor)]
    reader.wait_stream(builder)
    with torch.cuda.stream(reader):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        selection = torchbvh.select_blocks(tree, qpts, 4, query_offsets=query_offsets)
        torch.cuda._sleep(100_000_000)
        got = selection["block_indices"], torchbvh.attend_blocks(selection, q, k, v)
        del tree, selection
    with torch.cuda.stream(builder):
        over = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(8)]
    torch.cuda.synchronize()
    assert len(over) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed():
    """Forward and backward in one CUDA graph, replayed on new inputs; then a second graph."""
    scene = Scene("single", [1000], [500], 3, seed=21)
    selection = scene.select(5)
    sets = [_features(scene, BF16, 4, 4, 32, 8, seed=30 + i) for i in range(2)]
    want = [_run(scene, selection, f) for f in sets]
    for order in ((0, 1), (1, 0)):
        static = {x: scene.tensor(sets[0][x]).clone() for x in ("q", "k", "v", "grad")}
        table, edges = sets[0]["table"].cuda(), sets[0]["edges"].cuda()
        leaves = [static["q"], static["k"], static["v"], table]

        def step():
            fresh = [x.detach().requires_grad_(True) for x in leaves]
            out = torchbvh.attend_blocks(selection, *fresh[:3], bias_table=fresh[3], bias_edges=edges)
            return (out.detach(), *torch.autograd.grad(out, fresh, static["grad"]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step()
        for i in order:
            for x in ("q", "k", "v", "grad"):
                static[x].copy_(scene.tensor(sets[i][x]))
            table.copy_(sets[i]["table"])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want[i], results))


def test_selection_captured_and_replayed():
    scene = Scene("single", [2000], [300], 3, seed=22)
    queries = scene.tensor(scene.qpts)
    torchbvh.select_blocks(scene.bvh, queries, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        selection = torchbvh.select_blocks(scene.bvh, queries, 6)
    rng = np.random.default_rng(3)
    for _ in range(2):
        scene.qpts[0] = rng.random((300, 3), dtype=np.float32)
        queries.copy_(torch.as_tensor(scene.qpts[0]))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = oracle.select(scene.points[0], scene.orders[0], scene.qpts[0], 6)
        assert np.array_equal(selection["block_indices"].cpu().numpy(), want)


# ---------------------------------------------------------------------------
# Distance bias
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("num_buckets", [1, 2, 9, 32, 64])
@pytest.mark.parametrize("k", [1, 4, 7, 16, 32])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("per_head", [True, False])
def test_distance_bias(per_head, heads, k, num_buckets):
    g = torch.Generator().manual_seed(heads * 100 + k)
    shape = (2, 333, heads, k) if per_head else (2, 333, k)
    d2 = torch.rand(shape, generator=g) ** 3
    edges = torch.sort(torch.rand(num_buckets - 1, generator=g) ** 3).values
    if num_buckets > 2:
        d2[0, 0] = edges[1]  # exactly on a border: above it
        edges = edges[torch.randperm(num_buckets - 1, generator=g)]
    d2.view(-1)[:4] = torch.tensor([0.0, -1.0, float("nan"), float("inf")])[: d2.numel()]
    table = torch.randn((heads, num_buckets), generator=g)
    grad = torch.randn((2, 333, heads, k), generator=g)
    leaf = table.cuda().requires_grad_(True)
    out = torchbvh.distance_bias(d2.cuda(), leaf, edges.cuda())
    full = d2 if per_head else d2.unsqueeze(2).expand(2, 333, heads, k)
    bucket = oracle.buckets(full, edges)
    head = torch.arange(heads)[:, None]
    assert torch.equal(out.detach().cpu(), table[head, bucket])
    out.backward(grad.cuda())
    flat = (head * num_buckets + bucket).reshape(-1)
    total = lambda w: torch.zeros(heads * num_buckets, dtype=torch.float64).index_add_(0, flat, w.double().reshape(-1)).view(heads, -1)
    # Each term meets at most 700 float32 additions (a thread's column, the lanes, the warps), then 64 bits.
    oracle.within(leaf.grad, total(grad), (700 * 2.0**-24) * total(grad.abs()) + 1e-30, "grad of table")
    again = torch.autograd.grad(torchbvh.distance_bias(d2.cuda(), leaf, edges.cuda()), leaf, grad.cuda())[0]
    assert torch.equal(again, leaf.grad)


def test_distance_bias_of_nothing_and_strided():
    table = torch.randn((3, 5), device="cuda", requires_grad=True)
    edges = torch.linspace(0.1, 0.9, 4, device="cuda")
    out = torchbvh.distance_bias(torch.zeros((0, 4, 8), device="cuda"), table, edges)
    assert out.shape == (0, 4, 3, 8)
    out.sum().backward()
    assert not table.grad.any()
    d2 = torch.rand((2, 40, 12, 3), device="cuda").transpose(2, 3)[..., 1:9]
    assert torch.equal(torchbvh.distance_bias(d2, table, edges), torchbvh.distance_bias(d2.contiguous(), table, edges))


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

def test_a_point_transformer_step():
    """Build, select, two layers of attention, and a learned interpolation over displaced
    neighbours, all trained in one backward pass."""
    torch.manual_seed(0)
    batch, n, heads, channels = 2, 600, 4, 16
    pos = torch.rand((batch, n, 3), device="cuda")
    x = torch.randn((batch, n, heads * channels), device="cuda")
    weights = [torch.randn((heads * channels, 3 * heads * channels), device="cuda").mul_(0.1).requires_grad_(True)
               for _ in range(2)]
    table = torch.zeros((heads, 16), device="cuda", requires_grad=True)
    near = torch.zeros((heads, 16), device="cuda", requires_grad=True)
    edges = torch.logspace(-4, -1, 15, device="cuda")
    with torchbvh.BVH(pos) as bvh:
        selection = bvh.select_blocks(pos, 4)
        for w in weights:
            q, k, v = (x @ w).view(batch, n, 3, heads, channels).unbind(2)
            x = x + torchbvh.attend_blocks(selection, q, k, v, bias_table=table, bias_edges=edges).flatten(2)
    values = x.view(batch, n, heads, channels)
    moved = pos[:, :, None] + 0.02 * torch.randn((batch, n, heads, 3), device="cuda")
    idx, d2, _ = torchbvh.query_displaced_knn(pos, moved, 8)
    mix = torch.softmax(torchbvh.distance_bias(d2, near, edges), -1)
    out = torch.einsum("bnhkc,bnhk->bnhc", torchbvh.gather_neighbor_values(values, idx), mix)
    out.square().mean().backward()
    for p in (*weights, table, near):
        assert p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any())
    assert torchbvh.device_status() == 0
