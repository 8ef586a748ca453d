"""Attention over nearby blocks of points, and a learned bias by distance.

No counterpart in the reference, whose multi-head helpers weigh neighbours by
their inverse distance (torchbvh/_multihead.py:151-190). Here the weights are
learned:

* ``select_blocks`` chooses, for every query point, the ``num_blocks`` blocks of
  the BVH that are nearest to it. A block is a run of 64 consecutive points of
  the BVH's order (``sorted_indices``), its score the squared distance to the
  block's bounding box.
* ``attend_blocks`` is multi-head softmax attention of each query over the points
  of its blocks, optionally with a learned bias by distance bucket, with
  gradients for queries, keys, values and the bias table.
* ``distance_bias`` is the same bias for the neighbour lists of ``query_knn`` and
  ``query_displaced_knn``.

One selection serves any number of layers, heads and feature types over the
same points.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _native
from ._constants import (
    BLOCK_SIZE,
    MAX_BIAS_BUCKETS,
    MAX_BLOCK_CHANNELS,
    MAX_BLOCK_HEADS,
    MAX_SELECTED_BLOCKS,
    MAX_SHARED_HEADS,
)
from ._handles import (
    BVHHandle,
    BatchedBVHHandle,
    RaggedBVHHandle,
    _Handle,
    _batched_bvh_data,
    _bvh_data,
    _ragged_bvh_data,
)
from ._native import _C
from ._validation import (
    _as_contiguous,
    _as_contiguous_int64,
    _reject_unless,
    _validate_cuda_float32,
    _validate_offsets,
)

__all__ = ["BlockSelection", "select_blocks", "attend_blocks", "distance_bias"]

_SMALL = 16384  # queries of one cloud up to which the selection puts them in order itself


class BlockSelection(_Handle):
    """The blocks that ``select_blocks`` chose: a mapping with ``block_indices``
    (int64, -1 in empty slots), ``squared_distances`` (float32, ascending,
    FLT_MAX in empty slots), ``num_blocks`` and ``block_size``, and the plan that
    ``attend_blocks`` reads. It keeps what it needs of the BVH and of the query
    points: both may be destroyed or changed afterwards."""

    kind_message = "Block selection has been destroyed"
    marker = "_block_selection"

    def __init__(self, fields, geometry, keep, key_shape, query_shape):
        super().__init__(fields)
        self._geometry = geometry
        self._keep = keep  # tensors and host tables behind the geometry's pointers
        self._key_shape = key_shape      # leading shape of keys and values
        self._query_shape = query_shape  # leading shape of queries
        self._device = fields["block_indices"].device
        self._stream = _native.raw_stream(self._device) if self._device.type == "cuda" else None

    @property
    def device(self) -> torch.device:
        self._live_fields()
        return self._device

    def destroy(self) -> None:
        self._geometry = None
        self._keep = ()
        super().destroy()

    def _used_here(self) -> None:
        """Tells the allocator that the current stream reads the selection's memory. (The stream
        that made the selection is known to it: ``select_blocks`` recorded the tree's memory.)"""
        _record_use(self._keep, self._stream, self._device)


def _record_use(items, known: int | None, device: torch.device) -> None:
    """Tells the allocator that the current stream reads the tensors of ``items``, which lie in
    memory of the stream ``known`` (None: not known). A captured graph outlives any such record:
    there the memory has to be kept."""
    if _native.raw_stream(device) != known and not torch.cuda.is_current_stream_capturing():
        stream = torch.cuda.current_stream(device)
        for item in items:
            if isinstance(item, torch.Tensor) and item.is_cuda:
                item.record_stream(stream)


# The messages are put together only for a call that is refused.

def _check_query_points(query_points: torch.Tensor, rank: int, dim: int, device: torch.device) -> torch.Tensor:
    prefix = "select_blocks"
    if query_points.dim() != rank:
        raise ValueError(f"{prefix}: query_points must have shape {'(M, D)' if rank == 2 else '(B, M, D)'}")
    if query_points.size(-1) != dim:
        raise ValueError(f"{prefix}: query_points last dimension must match BVH dim")
    _validate_cuda_float32(prefix, query_points, "query_points")
    if query_points.device != device:
        raise ValueError(f"{prefix}: query_points must be on the same device as the BVH")
    if query_points.numel() // dim > 2**31 - 1:
        raise ValueError(f"{prefix}: total query count must fit in signed int32")
    return _as_contiguous(query_points.detach())


def select_blocks(bvh: BVHHandle | BatchedBVHHandle | RaggedBVHHandle, query_points: torch.Tensor, num_blocks: int, *,
                  query_offsets: torch.Tensor | None = None, backward: bool = True) -> BlockSelection:
    """Chooses for every query the ``num_blocks`` (1 to 32) blocks of 64 points
    whose bounding boxes are nearest, by (squared distance, block index).

    Dispatches on the handle like ``query_knn``: query points ``(M, D)``,
    ``(B, M, D)``, or packed ``(total_M, D)`` with ``query_offsets`` for a ragged
    BVH. ``block_indices`` and ``squared_distances`` have the queries' leading
    shape and ``num_blocks`` last; block ``j`` holds the points
    ``sorted_indices[64 * j : 64 * (j + 1)]`` of the query's cloud. Slots past the
    cloud's last block, and all slots of a query that is not finite, hold -1 and
    FLT_MAX. Clouds may be smaller than a block.

    ``backward=False`` leaves out the lists that the backward pass of
    ``attend_blocks`` needs, for inference. Carries no gradient.
    """
    prefix = "select_blocks"
    if not (isinstance(num_blocks, int) and not isinstance(num_blocks, bool) and 1 <= num_blocks <= MAX_SELECTED_BLOCKS):
        raise ValueError(f"{prefix}: num_blocks must be 1 to {MAX_SELECTED_BLOCKS}")
    geometry = _native.BlockGeometry(num_blocks=num_blocks, backward=1 if backward else 0)
    if isinstance(bvh, RaggedBVHHandle):
        _reject_unless(query_offsets is not None, f"{prefix}: query_offsets is required for a ragged BVH")
        data, tree = _ragged_bvh_data(bvh, prefix)
        device = tree["node_aabbs"].device
        queries = _check_query_points(query_points, 2, tree["dim"], device)
        query_offsets = _as_contiguous_int64(query_offsets)
        host = _validate_offsets(prefix, query_offsets, total_rows=int(queries.size(0)), device=device)
        _reject_unless(len(host) - 1 == data["batch_size"], f"{prefix}: query_offsets batch size must match BVH batch_size")
        table = _native.block_table(tree["point_offsets"], host)
        table_dev = torch.tensor(list(table), dtype=torch.int64, device=device)
        geometry.num_clouds, geometry.table_host, geometry.table_dev = (
            len(host) - 1, ctypes.cast(table, ctypes.c_void_p), table_dev.data_ptr())
        order = None
        if max(b - a for a, b in zip(host, host[1:])) > _SMALL:
            order = _native.keeps_device(_C.morton_sort_queries_ragged)(
                queries, query_offsets, int(queries.size(0)), tree["scene_min"], tree["scene_max"])
        keep = (table, table_dev)
        key_shape = (tree["point_offsets"][-1],)
    else:
        if query_offsets is not None:
            raise TypeError(f"{prefix}: query_offsets requires a RaggedBVHHandle")
        batched = isinstance(bvh, BatchedBVHHandle)
        tree = _batched_bvh_data(bvh, prefix) if batched else _bvh_data(bvh, prefix)
        device = tree["node_aabbs"].device
        queries = _check_query_points(query_points, 3 if batched else 2, tree["dim"], device)
        clouds, per_cloud = (int(queries.size(0)) if batched else 1), int(queries.size(-2))
        _reject_unless(not batched or clouds == tree["batch_size"],
                       f"{prefix}: query_points batch size must match BVH batch_size")
        geometry.num_clouds, geometry.points_per_cloud, geometry.queries_per_cloud = (
            clouds, tree["num_leaves"], per_cloud)
        order = None
        if per_cloud > _SMALL:
            lift = (lambda t: t) if batched else (lambda t: t.unsqueeze(0))
            order = _native.keeps_device(_C.morton_sort_queries_narrow)(
                lift(queries), lift(tree["scene_min"]), lift(tree["scene_max"]))
        keep = ()
        key_shape = ((clouds,) if batched else ()) + (tree["num_leaves"],)
    nodes, leaves = tree["node_aabbs"], tree["sorted_indices"]
    # The caller may drop the tree as soon as this returns, and with it memory of the stream that built it.
    _record_use((nodes, leaves, tree["scene_min"], tree["scene_max"]), bvh._built_on, device)
    geometry.device, geometry.dim = device.index, tree["dim"]
    geometry.node_aabbs, geometry.sorted_indices = nodes.data_ptr(), leaves.data_ptr()
    geometry.query_points = queries.data_ptr()
    geometry.order = None if order is None else order.data_ptr()
    lead = tuple(queries.shape[:-1])
    blocks, distances, plan = _native.select_blocks(geometry, queries.numel() // tree["dim"], device)
    fields = {"block_indices": blocks.view(*lead, num_blocks), "squared_distances": distances.view(*lead, num_blocks),
              "num_blocks": num_blocks, "block_size": BLOCK_SIZE}
    return BlockSelection(fields, geometry, (nodes, leaves, plan, *keep), key_shape, lead)


def _check_bias(prefix: str, table: torch.Tensor, edges: torch.Tensor, heads: int | None, device: torch.device,
                table_name: str, edges_name: str) -> None:
    if table.dim() != 2 or (heads is not None and table.size(0) != heads):
        raise ValueError(f"{prefix}: {table_name} must have shape (H, num_buckets)")
    buckets = table.size(1)
    if not 1 <= buckets <= MAX_BIAS_BUCKETS:
        raise ValueError(f"{prefix}: {table_name} must have 1 to {MAX_BIAS_BUCKETS} buckets")
    if edges.dim() != 1 or edges.size(0) != buckets - 1:
        raise ValueError(f"{prefix}: {edges_name} must have shape (num_buckets - 1,)")
    _validate_cuda_float32(prefix, table, table_name)
    _validate_cuda_float32(prefix, edges, edges_name)
    if table.device != device or edges.device != device:
        raise ValueError(f"{prefix}: {table_name} and {edges_name} must be on the same device as the other inputs")


def _refuse_tangents(prefix: str, *tensors: torch.Tensor | None) -> None:
    """Forward-mode derivatives would be dropped: a dual tensor need not require a gradient."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{prefix}: forward-mode derivatives are not implemented")


class _AttendBlocks(torch.autograd.Function):
    """Attention with the backward pass of the native library. Keeps its inputs,
    its output and two numbers a row (its softmax's maximum and sum). Where a bias
    table trains with 16-bit features the kept output is float32: the table's
    gradient sums float32 terms whose errors would otherwise all lean with the
    rounding of their row's output."""

    @staticmethod
    def forward(ctx, queries, keys, values, table, edges, selection, scale):
        geometry = selection._geometry
        exactly = ctx.needs_input_grad[3] and queries.dtype != torch.float32
        out, stats, exact = _native.attend_blocks(geometry, queries, keys, values, table, edges, scale, True, exactly)
        ctx.save_for_backward(queries, keys, values, table, edges, None if exactly else out, exact, stats)
        ctx.selection, ctx.geometry, ctx.keep, ctx.scale = selection, geometry, selection._keep, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        queries, keys, values, table, edges, out, exact, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if ctx.selection._alive:
            ctx.selection._used_here()
        grads = _native.attend_blocks_backward(ctx.geometry, queries, keys, values, table, edges, ctx.scale, out,
                                               exact, stats, _as_contiguous(grad_out), need[0], need[1] or need[2],
                                               need[3] and table is not None)
        return (*(g if wanted else None for g, wanted in zip(grads, need)), None, None, None)


def attend_blocks(selection: BlockSelection, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, *,
                  bias_table: torch.Tensor | None = None, bias_edges: torch.Tensor | None = None,
                  scale: float | None = None) -> torch.Tensor:
    """Multi-head attention of every query over the points of its selected blocks.

    ``queries (M, H, C)``, ``keys`` and ``values (N, Hkv, C)`` in the caller's
    point order for a single cloud; ``(B, M, H, C)`` and ``(B, N, Hkv, C)`` for a
    fixed-size batch; packed like the points and query points for a ragged one.
    float32, float16 or bfloat16, all of one type; ``C`` is 1 to 128, ``H`` a
    multiple of ``Hkv`` (query heads ``h`` of one run of ``H / Hkv`` share a
    key/value head). Returns the shape and type of ``queries``.

    For query ``i`` and head ``h`` the logit of point ``j`` is
    ``scale * <queries[i, h], keys[j, h // (H / Hkv)]>`` (``scale`` defaults to
    ``C ** -0.5``), plus ``bias_table[h, b]`` where ``b`` is the number of
    ``bias_edges`` not above the squared distance of the two points (float32).
    ``bias_table (H, num_buckets)`` and ``bias_edges (num_buckets - 1,)`` are
    float32, with 1 to 64 buckets; a bias of -inf masks its bucket, whose points
    still have to be finite (they enter with a weight of zero). A query with no
    point to attend to gets zeros.

    Differentiable in ``queries``, ``keys``, ``values`` and ``bias_table`` (the
    selection must have been made with ``backward=True``), in reverse mode. Results and gradients
    of equal inputs are equal bit for bit: nothing is summed in changing order.
    (A call of more queries, or a larger batch, may split its sums otherwise.)

    All sums and the softmax are float32. With 16-bit features the weights are
    rounded to 16 bits before their product with the values, and so are the
    logits' gradients before theirs with keys and queries: one more half step of
    the type, relative to each (float16: of weights down to 2^-29, and of
    gradients down to 2^-29 of the largest that they could be; below, 2^-40 of
    it). Products of float32 features keep all but 2^-22 of themselves. The
    table's gradient is summed in float32 within a thread block, in float64
    across them.
    """
    prefix = "attend_blocks"
    if not isinstance(selection, BlockSelection):
        raise TypeError(f"{prefix}: selection must be a BlockSelection returned by select_blocks")
    device = selection.device
    query_shape, key_shape = selection._query_shape, selection._key_shape
    if queries.dim() != len(query_shape) + 2 or tuple(queries.shape[:-2]) != query_shape:
        raise ValueError(f"{prefix}: queries must have shape {(*query_shape, 'H', 'C')}".replace("'", ""))
    heads, channels = queries.shape[-2:]
    for name, t in (("keys", keys), ("values", values)):
        if t.dim() != len(key_shape) + 2 or tuple(t.shape[:-2]) != key_shape or t.size(-1) != channels:
            raise ValueError(f"{prefix}: {name} must have shape {(*key_shape, 'Hkv', 'C')}".replace("'", ""))
    key_heads = keys.size(-2)
    if key_heads != values.size(-2):
        raise ValueError(f"{prefix}: keys and values must have the same heads")
    if heads < 1 or key_heads < 1 or heads % key_heads != 0:
        raise ValueError(f"{prefix}: query heads must be a multiple of key heads")
    if heads // key_heads > MAX_SHARED_HEADS or heads > MAX_BLOCK_HEADS:
        raise ValueError(f"{prefix}: at most {MAX_BLOCK_HEADS} query heads, and {MAX_SHARED_HEADS} to a key head")
    if not 1 <= channels <= MAX_BLOCK_CHANNELS:
        raise ValueError(f"{prefix}: channels must be 1 to {MAX_BLOCK_CHANNELS}")
    dtype = queries.dtype
    for name, t in (("queries", queries), ("keys", keys), ("values", values)):
        if not t.is_cuda:
            raise ValueError(f"{prefix}: {name} must be a CUDA tensor")
        if t.device != device:
            raise ValueError(f"{prefix}: {name} must be on the same device as the selection")
        if t.dtype != dtype or dtype not in _native._FEATURE_TYPES:
            raise ValueError(f"{prefix}: queries, keys and values must share one type: float32, float16 or bfloat16")
    if (bias_table is None) != (bias_edges is None):
        raise ValueError(f"{prefix}: bias_table and bias_edges must be given together")
    if bias_table is not None:
        _check_bias(prefix, bias_table, bias_edges, heads, device, "bias_table", "bias_edges")
        bias_table, bias_edges = _as_contiguous(bias_table), _as_contiguous(bias_edges.detach())
    scale = channels**-0.5 if scale is None else float(scale)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"{prefix}: scale must be finite in float32")
    _refuse_tangents(prefix, queries, keys, values, bias_table)
    queries, keys, values = _as_contiguous(queries), _as_contiguous(keys), _as_contiguous(values)
    selection._used_here()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (queries, keys, values, bias_table)):
        if not selection._geometry.backward:
            raise ValueError(f"{prefix}: gradients need a selection made with backward=True")
        return _AttendBlocks.apply(queries, keys, values, bias_table, bias_edges, selection, scale)
    return _native.attend_blocks(selection._geometry, queries, keys, values, bias_table, bias_edges, scale, False,
                                 False)[0]


class _DistanceBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, squared_distances, table, edges, per_head):
        ctx.save_for_backward(squared_distances, edges)
        ctx.heads, ctx.per_head = int(table.size(0)), per_head
        return _native.distance_bias(squared_distances, ctx.heads, per_head, table, edges)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        squared_distances, edges = ctx.saved_tensors
        grad = _native.distance_bias_backward(squared_distances, ctx.heads, ctx.per_head, edges, _as_contiguous(grad_out))
        return None, grad, None, None


def distance_bias(squared_distances: torch.Tensor, table: torch.Tensor, edges: torch.Tensor) -> torch.Tensor:
    """Learned bias of neighbour lists by distance bucket:
    ``out[b, i, h, j] = table[h, n]``, ``n`` the number of ``edges`` not above
    the squared distance (a NaN distance counts none).

    ``squared_distances (B, N, H, k)`` (one list a head, as from
    ``query_displaced_knn``) or ``(B, N, k)`` (as from ``query_knn``, shared by
    the heads) float32; ``table (H, num_buckets)`` float32 with 1 to 64 buckets;
    ``edges (num_buckets - 1,)`` float32, in any order. Returns
    ``(B, N, H, k)`` float32, differentiable in ``table``, in reverse mode; its
    gradient is summed in a fixed order.
    """
    prefix = "distance_bias"
    rank = squared_distances.dim()
    if rank not in (3, 4):
        raise ValueError(f"{prefix}: squared_distances must have shape (B, N, H, k) or (B, N, k)")
    _validate_cuda_float32(prefix, squared_distances, "squared_distances")
    _check_bias(prefix, table, edges, None, squared_distances.device, "table", "edges")
    heads = table.size(0)
    if rank == 4 and squared_distances.size(2) != heads:
        raise ValueError(f"{prefix}: squared_distances head dimension must match table")
    if not 1 <= heads <= MAX_BLOCK_HEADS:
        raise ValueError(f"{prefix}: table must have at least one head, and at most {MAX_BLOCK_HEADS}")
    _refuse_tangents(prefix, table)
    squared_distances = _as_contiguous(squared_distances.detach())
    table, edges = _as_contiguous(table), _as_contiguous(edges.detach())
    if torch.is_grad_enabled() and table.requires_grad:
        return _DistanceBias.apply(squared_distances, table, edges, rank == 4)
    return _native.distance_bias(squared_distances, heads, rank == 4, table, edges)
