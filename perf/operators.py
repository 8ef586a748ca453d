"""Cases that measure block selection, block attention and the distance bias.

``run`` computes each operator in plain torch operations, or, where ``own`` is
true, with the package's calls. A case is one pass of one operator:

- ``select``: for every query point, the blocks of 64 consecutive leaves of a
  cloud's Morton order whose boxes are nearest;
- ``attend``: multi-head softmax attention of every query over the points of its
  selected blocks, with a learned bias by distance bucket; with ``train`` also
  the gradients of queries, keys, values and the bias table;
- ``bias``: the same bias for k-NN squared distances, with ``train`` the
  gradient of its table.

Clouds hold the corners 0 and 1 of their unit box, so that the Morton cell of a
point is ``floor(p * bins)`` without rounding in any arithmetic.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64
FAR = float(np.finfo(np.float32).max)


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def _select(name, layout, sizes, queries, dim, n, cloud, train):
    return {"name": name, "op": "select", "layout": layout, "sizes": sizes, "queries": queries, "dim": dim, "blocks": n,
            "cloud": cloud, "train": train}


def _attend(name, layout, sizes, queries, dim, n, cloud, train, dtype, heads, kv_heads, channels, buckets):
    return {"name": name, "op": "attend", "layout": layout, "sizes": sizes, "queries": queries, "dim": dim, "blocks": n,
            "cloud": cloud, "train": train, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "channels": channels, "buckets": buckets}


def _bias(name, points, heads, k, per_head, buckets, train):
    return {"name": name, "op": "bias", "points": points, "heads": heads, "k": k, "per_head": per_head,
            "buckets": buckets, "train": train}


def listed():
    """``sizes`` is one cloud size, ``BxN``, or a comma list of ragged sizes; ``queries`` the same
    for the query points, or ``self`` where the points query themselves."""
    return [
        # One new query against a kept cloud: an interactive probe, all latency.
        _select("select one query", "single", "4096", "1", 3, 8, "uniform", False),
        # The 10,000-point cloud of the benchmark's first workload, every point of a second cloud asking.
        _select("select 10k", "single", "10000", "10000", 3, 8, "uniform", False),
        # The benchmark's clustered batch (16 x 65,536, displaced self-queries), selected for training.
        _select("select 16x65k train", "batched", "16x65536", "self", 3, 16, "clusters", True),
        # One probe of a deployed model: a single token over 16 blocks, all latency.
        _attend("attend one query bf16", "single", "10000", "1", 3, 16, "uniform", False, "bfloat16", 8, 8, 64, 32),
        # Inference on packed clouds of very different sizes, an odd channel count.
        _attend("attend ragged fp16", "ragged", "1024,1531,17000,2750,9001,64,4099", "self", 3, 8, "uniform", False,
                "float16", 6, 6, 24, 16),
        # Inference on a batch, the largest forward pass.
        _attend("attend 4x16k bf16", "batched", "4x16384", "self", 3, 8, "clusters", False, "bfloat16", 4, 4, 32, 32),
        # A training step of a point transformer layer.
        _attend("attend train 16k bf16", "single", "16384", "self", 3, 8, "uniform", True, "bfloat16", 8, 8, 32, 32),
        # Training with shared key/value heads and no bias, wider heads, 2-D points.
        _attend("attend train shared bf16", "batched", "2x8192", "self", 2, 8, "uniform", True, "bfloat16", 8, 2, 64, 0),
        # The package's own type, odd sizes everywhere.
        _attend("attend train fp32", "batched", "3x2501", "1999", 3, 5, "clusters", True, "float32", 3, 3, 20, 9),
        # Bias of the k-NN lists of a clustered batch, one list a head (displaced queries), training.
        _bias("bias train 262k per head", 262144, 4, 16, True, 32, True),
        # Bias of shared lists broadcast over the heads.
        _bias("bias 100k shared", 100000, 8, 16, False, 32, False),
        _bias("bias 500 shared", 500, 3, 4, False, 9, False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["select", "attend", "attend", "bias"])
    if op == "bias":
        heads, k = rng.choice([1, 2, 3, 4, 8]), rng.choice([4, 8, 16, 32])
        case = _bias("", _spread(rng, 200, 16_000_000 // (heads * k)), heads, k, rng.random() < 0.5,
                     rng.randint(2, 48), rng.random() < 0.5)
        del case["name"]
        return case
    layout = rng.choice(["single", "batched", "ragged"])
    dim, n, train = rng.choice([2, 3]), rng.randint(1, 24), rng.random() < 0.5
    cloud = rng.choice(["uniform", "clusters"])
    if op == "select":
        total = _spread(rng, 300, 200_000)
    else:
        heads = rng.choice([1, 2, 3, 4, 6, 8])
        kv_heads = rng.choice([h for h in (1, 2, 3, 4, 6, 8) if heads % h == 0])
        channels = rng.choice([8, 12, 16, 24, 32, 40, 48, 64, 80, 128])
        n = min(n, 12)
        total = _spread(rng, 300, max(400, min(40_000, 1_000_000_000 // (n * BLOCK * heads * channels))))
    clouds = 1 if layout == "single" else rng.randint(2, 5)
    if layout == "single":
        sizes, queries = str(total), "self" if rng.random() < 0.5 else str(_spread(rng, 1, total))
    elif layout == "batched":
        each = max(2, total // clouds)
        sizes, queries = "%dx%d" % (clouds, each), "self" if rng.random() < 0.5 else str(_spread(rng, 1, each))
    else:
        part = [rng.uniform(0.1, 1.0) for _ in range(clouds)]
        sizes, queries = ",".join(str(max(2, int(total * p / sum(part)))) for p in part), "self"
    if op == "select":
        case = _select("", layout, sizes, queries, dim, n, cloud, train)
    else:
        case = _attend("", layout, sizes, queries, dim, n, cloud, train, rng.choice(["float32", "bfloat16", "float16"]),
                       heads, kv_heads, channels, rng.choice([0, 2, 9, 16, 32, 48]))
    del case["name"]
    return case


def _sizes(case):
    """Points and queries of each cloud."""
    text = case["sizes"]
    if case["layout"] == "batched":
        b, n = (int(v) for v in text.split("x"))
        points = [n] * b
    else:
        points = [int(v) for v in text.split(",")]
    queries = list(points) if case["queries"] == "self" else [int(case["queries"])] * len(points)
    return points, queries


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _edges(buckets):
    """Bucket borders of squared distances: doubling from small to the size of the unit box."""
    if buckets < 2:
        return torch.empty(0, device="cuda")
    return torch.logspace(-5, -1, buckets - 1, base=10.0, dtype=torch.float64).float().cuda()


def _cloud(g, n, dim, kind):
    if kind == "uniform":
        p = torch.rand((n, dim), generator=g, device="cuda")
    else:
        centres = torch.rand((32, dim), generator=g, device="cuda")
        which = torch.randint(0, 32, (n,), generator=g, device="cuda")
        p = (centres[which] + 0.02 * torch.randn((n, dim), generator=g, device="cuda")).clamp(0, 1)
    p[0] = 0
    p[-1] = 1
    return p


def _geometry(case, g):
    points, queries = _sizes(case)
    p = torch.cat([_cloud(g, n, case["dim"], case["cloud"]) for n in points])
    if case["queries"] == "self":
        q = p + 0.01 * torch.randn(p.shape, generator=g, device="cuda")
    else:
        q = torch.rand((sum(queries), case["dim"]), generator=g, device="cuda")
    return p, q


def _features(case, g, total_points, total_queries):
    dtype = getattr(torch, case["dtype"])
    h, kv, c = case["heads"], case["kv_heads"], case["channels"]
    out = {
        "q": torch.randn((total_queries, h, c), generator=g, device="cuda").to(dtype),
        "k": torch.randn((total_points, kv, c), generator=g, device="cuda").to(dtype),
        "v": torch.randn((total_points, kv, c), generator=g, device="cuda").to(dtype),
        "table": None, "edges": None, "grad": None,
    }
    if case["buckets"]:
        # A learned bias falls with the distance and differs by head.
        slope = torch.linspace(0, -2, case["buckets"], device="cuda")
        out["table"] = slope + 0.5 * torch.randn((h, case["buckets"]), generator=g, device="cuda")
        out["edges"] = _edges(case["buckets"])
    if case["train"]:
        out["grad"] = torch.randn((total_queries, h, c), generator=g, device="cuda").to(dtype)
    return out


def _bias_inputs(case, g):
    shape = (1, case["points"]) + ((case["heads"],) if case["per_head"] else ()) + (case["k"],)
    # Squared distances of ascending neighbours in a unit box.
    near = torch.rand(shape, generator=g, device="cuda").cumsum(-1) * 0.01
    state = {"d2": near * near, "edges": _edges(case["buckets"]),
             "table": torch.randn((case["heads"], case["buckets"]), generator=g, device="cuda"), "grad": None}
    if case["train"]:
        state["grad"] = torch.randn((1, case["points"], case["heads"], case["k"]), generator=g, device="cuda")
    return state


def _offsets(sizes):
    return torch.tensor([0] + sizes, device="cuda").cumsum(0)


def _shaped(case, packed, sizes):
    """A packed tensor in the case's layout: (N, ...), (B, N, ...) or packed."""
    return packed.view(len(sizes), sizes[0], *packed.shape[1:]) if case["layout"] == "batched" else packed


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "bias":
        state = {"case": case, **_bias_inputs(case, g)}
        if own and case["train"]:
            state["table"].requires_grad_(True)
        return state
    points, queries = _sizes(case)
    p, q = _geometry(case, g)
    state = {"case": case, "points": p, "query_points": q}
    if case["op"] == "attend":
        state.update(_features(case, g, sum(points), sum(queries)))
    if own:
        import torchbvh_b200

        ragged = case["layout"] == "ragged"
        state["query_points"] = _shaped(case, q, queries)
        state["offsets"] = _offsets(queries) if ragged else None
        state["bvh"] = torchbvh_b200.BVH(_shaped(case, p, points), batch_offsets=_offsets(points) if ragged else None)
        if case["op"] == "attend":
            # A program keeps the selection: all layers of a model over one cloud use it.
            state["selection"] = state["bvh"].select_blocks(state["query_points"], case["blocks"],
                                                            query_offsets=state["offsets"], backward=case["train"])
            for name, sizes in (("q", queries), ("k", points), ("v", points), ("grad", queries)):
                if state[name] is not None:
                    state[name] = _shaped(case, state[name], sizes)
            if case["train"]:
                for name in ("q", "k", "v") + (("table",) if case["buckets"] else ()):
                    state[name].requires_grad_(True)
        return state
    state["cloud_of_query"] = torch.repeat_interleave(torch.arange(len(queries), device="cuda"),
                                                      torch.tensor(queries, device="cuda"))
    state["starts"], state["counts"] = _offsets(points)[:-1], torch.tensor(points, device="cuda")
    state["leaves"] = _plain_leaves(state)
    state["boxes"] = _plain_boxes(state)
    if case["op"] == "attend":
        state["selected"] = _plain_select(state)[0]
    return state


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------

def _plain_leaves(state):
    """Packed point rows in each cloud's Morton order (stable)."""
    p, dim = state["points"], state["points"].shape[1]
    bits = 10 if dim == 3 else 16
    cell = (p * 2 ** bits).long().clamp(0, 2 ** bits - 1)
    step = torch.arange(bits, device="cuda")
    spread = ((cell[:, :, None] >> step) & 1) << (step * dim)
    code = sum(spread[:, a].sum(-1) << a for a in range(dim))
    cloud = torch.repeat_interleave(torch.arange(len(state["counts"]), device="cuda"), state["counts"])
    return torch.sort((cloud << 32) | code, stable=True).indices


def _plain_boxes(state):
    """Lower and upper corners (clouds, blocks, D); blocks past a cloud's end are infinitely far."""
    nb = (state["counts"] + BLOCK - 1) // BLOCK
    block = torch.arange(int(nb.max()), device="cuda")
    leaf = block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    leaf = torch.minimum(leaf[None], state["counts"][:, None, None] - 1) + state["starts"][:, None, None]
    inside = state["points"][state["leaves"][leaf]]
    there = (block[None] < nb[:, None])[..., None]
    inf = torch.tensor(math.inf, device="cuda")
    return torch.where(there, inside.amin(2), inf), torch.where(there, inside.amax(2), inf)


def _plain_select(state):
    lo, hi = state["boxes"]
    cloud, q, n = state["cloud_of_query"], state["query_points"], state["case"]["blocks"]
    dist = 0
    for a in range(q.shape[1]):
        off = torch.maximum(lo[cloud, :, a] - q[:, a, None], (q[:, a, None] - hi[cloud, :, a]).clamp(min=0))
        dist = dist + off * off
    if dist.shape[1] < n:  # fewer blocks than asked for: the rest of the slots stays empty
        dist = torch.cat([dist, torch.full((len(q), n - dist.shape[1]), FAR, device="cuda")], 1)
    index = torch.arange(dist.shape[1], device="cuda")
    # (distance, block) pairs as whole numbers: ties go to the lowest block.
    pair = (dist.view(torch.int32).long() << 32) | index
    pair = torch.where(dist < FAR, pair, torch.iinfo(torch.int64).max)
    pair = torch.topk(pair, n, dim=1, largest=False, sorted=True).values
    empty = pair == torch.iinfo(torch.int64).max
    near = torch.where(empty, FAR, (pair >> 32).int().view(torch.float32))
    return torch.where(empty, -1, pair & 0xFFFFFFFF), near


def _plain_bucket(d2, edges):
    return (d2[..., None] >= edges).sum(-1)


def _plain_attend(state):
    case, sel = state["case"], state["selected"]
    h, kv, c = case["heads"], case["kv_heads"], case["channels"]
    q, k, v = (state[x].float() for x in ("q", "k", "v"))
    m, scale = q.shape[0], 1.0 / math.sqrt(c)
    count = state["counts"][state["cloud_of_query"]][:, None]
    leaf = (sel[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(m, -1)
    there = (sel >= 0).repeat_interleave(BLOCK, 1) & (leaf < count)
    leaf = torch.minimum(leaf.clamp(min=0), count - 1) + state["starts"][state["cloud_of_query"]][:, None]
    rows = state["leaves"][leaf]
    qg = q.view(m, kv, h // kv, c)
    ks, vs = k[rows].transpose(1, 2), v[rows].transpose(1, 2)  # (M, kv, S, C)
    z = (qg @ ks.transpose(2, 3)).view(m, h, -1) * scale
    if state["table"] is not None:
        off = state["points"][rows] - state["query_points"][:, None]
        d2 = off[..., 0] * off[..., 0]
        for a in range(1, off.shape[-1]):
            d2 = d2 + off[..., a] * off[..., a]
        bucket = _plain_bucket(d2, state["edges"])
        z = z + state["table"][:, bucket].transpose(0, 1)
    z = torch.where(there[:, None], z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top > -math.inf, top, 0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    pg = p.view(m, kv, h // kv, -1)
    out = (pg @ vs).view(m, h, c)
    if not case["train"]:
        return [out.to(state["q"].dtype)]
    do = state["grad"].float()
    dog = do.view(m, kv, h // kv, c)
    ds = pg * (dog @ vs.transpose(2, 3) - (dog * out.view_as(dog)).sum(-1, keepdim=True))
    dq = (ds @ ks).view(m, h, c) * scale
    dk = torch.zeros_like(k).index_add_(0, rows.reshape(-1), (ds.transpose(2, 3) @ qg).transpose(1, 2).reshape(-1, kv, c) * scale)
    dv = torch.zeros_like(v).index_add_(0, rows.reshape(-1), (pg.transpose(2, 3) @ dog).transpose(1, 2).reshape(-1, kv, c))
    dtype = state["q"].dtype
    grads = [dq.to(dtype), dk.to(dtype), dv.to(dtype)]
    if state["table"] is not None:
        # Sums of millions of terms: in 64 bits.
        dt = torch.zeros((case["buckets"], h), dtype=torch.float64, device="cuda")
        dt.index_add_(0, bucket.reshape(-1), ds.view(m, h, -1).transpose(1, 2).reshape(-1, h).double())
        grads.append(dt.T.float())
    return [out.to(dtype), *grads]


def _plain_bias(state):
    case = state["case"]
    bucket = _plain_bucket(state["d2"], state["edges"])
    if not case["per_head"]:
        bucket = bucket.unsqueeze(2).expand(-1, -1, case["heads"], -1)
    head = torch.arange(case["heads"], device="cuda")[:, None]
    out = state["table"][head, bucket]
    if not case["train"]:
        return [out]
    at = (head * case["buckets"] + bucket).reshape(-1)
    dt = torch.zeros(case["heads"] * case["buckets"], dtype=torch.float64, device="cuda")
    dt.index_add_(0, at, state["grad"].reshape(-1).double())
    return [out, dt.view_as(state["table"]).float()]


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def _run_own(state):
    import torchbvh_b200

    case = state["case"]
    if case["op"] == "select":
        selection = state["bvh"].select_blocks(state["query_points"], case["blocks"], query_offsets=state["offsets"],
                                               backward=case["train"])
        return [selection["block_indices"].reshape(-1, case["blocks"]),
                selection["squared_distances"].reshape(-1, case["blocks"])]
    if case["op"] == "bias":
        out = torchbvh_b200.distance_bias(state["d2"], state["table"], state["edges"])
        if not case["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, [state["table"]], state["grad"])]
    out = torchbvh_b200.attend_blocks(state["selection"], state["q"], state["k"], state["v"],
                                      bias_table=state["table"], bias_edges=state["edges"])
    packed = [out.detach().reshape(-1, case["heads"], case["channels"])]
    if not case["train"]:
        return packed
    leaves = [state["q"], state["k"], state["v"]] + ([state["table"]] if state["table"] is not None else [])
    grads = torch.autograd.grad(out, leaves, state["grad"])
    return packed + [x.reshape(-1, *x.shape[-2:]) for x in grads[:3]] + list(grads[3:])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_bias(state) if op == "bias" else _plain_attend(state) if op == "attend" else list(_plain_select(state))


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "bias":
        lists = case["points"] * case["k"] * (case["heads"] if case["per_head"] else 1)
        values = case["points"] * case["k"] * case["heads"]
        table = 4 * case["heads"] * case["buckets"] * (2 if case["train"] else 1)
        return {"bytes": 4 * (lists + values * (2 if case["train"] else 1)) + table, "flops": values}
    points, queries = _sizes(case)
    n, m, dim = sum(points), sum(queries), case["dim"]
    blocks = [(x + BLOCK - 1) // BLOCK for x in points]
    if case["op"] == "select":
        return {"bytes": 4 * dim * m + 8 * dim * sum(blocks) + 12 * case["blocks"] * m,
                "flops": sum(q * min(case["blocks"], b) * 5 * dim for q, b in zip(queries, blocks))}
    h, kv, c = case["heads"], case["kv_heads"], case["channels"]
    e = 4 if case["dtype"] == "float32" else 2
    seen = sum(q * min(case["blocks"] * BLOCK, x) for q, x in zip(queries, points))
    n = sum(min(x, q * case["blocks"] * BLOCK) for q, x in zip(queries, points))  # few queries read few points
    bytes_ = e * c * (2 * m * h + 2 * n * kv) + 8 * case["blocks"] * m + (4 * dim * (m + n) if case["buckets"] else 0)
    flops = 4 * seen * h * c
    if case["train"]:
        bytes_ += e * c * (2 * m * h + 2 * n * kv) + 8 * h * case["buckets"]
        flops += 10 * seen * h * c
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_order(points):
    """Rows of one cloud by Morton code, lowest row first among equals."""
    bins = 1024 if points.shape[1] == 3 else 65536
    cell = np.minimum(np.floor(points.astype(np.float64) * bins), bins - 1).astype(np.int64)
    code = np.zeros(len(points), np.int64)
    for bit in range(bins.bit_length() - 1):
        for axis in range(points.shape[1]):
            code |= ((cell[:, axis] >> bit) & 1) << (bit * points.shape[1] + axis)
    return np.argsort(code, kind="stable")


def _exact_blocks(points, order, queries, n):
    """Box distances of float32 arithmetic by its definition, on the host; the n nearest of each query."""
    first = np.arange(0, len(points), BLOCK)
    lo, hi = (f.reduceat(points[order], first, axis=0) for f in (np.minimum, np.maximum))
    chosen = np.full((len(queries), n), -1, np.int64)
    for at in range(0, len(queries), 8192):
        q = queries[at:at + 8192]
        d = np.zeros((len(q), len(first)), np.float32)
        for axis in range(points.shape[1]):
            gap = np.maximum(lo[None, :, axis] - q[:, None, axis], np.maximum(q[:, None, axis] - hi[None, :, axis], np.float32(0)))
            d += gap * gap
        take = min(n, len(first))
        chosen[at:at + 8192, :take] = np.argsort(d, axis=1, kind="stable")[:, :take]
    return chosen


def _exact_distances(case, p, q):
    """Distances of the selected blocks in 64 bits, from boxes of 64-bit coordinates."""
    out, p_at, q_at = [], 0, 0
    for np_, nq in zip(*_sizes(case)):
        pts, qs = p[p_at:p_at + np_], q[q_at:q_at + nq]
        order = _exact_order(pts)
        chosen = _exact_blocks(pts, order, qs, case["blocks"])
        first = np.arange(0, np_, BLOCK)
        lo, hi = (f.reduceat(pts[order], first, axis=0).astype(np.float64) for f in (np.minimum, np.maximum))
        gap = np.maximum(lo[chosen] - qs[:, None].astype(np.float64), qs[:, None].astype(np.float64) - hi[chosen])
        d = (np.maximum(gap, 0) ** 2).sum(-1)
        out.append(np.where(chosen < 0, FAR, d))
        p_at, q_at = p_at + np_, q_at + nq
    return torch.from_numpy(np.concatenate(out))


def _exact_attend(case, g):
    p, q = _geometry(case, g)
    points, queries = _sizes(case)
    f = _features(case, g, sum(points), sum(queries))
    h, kv, c = case["heads"], case["kv_heads"], case["channels"]
    group = torch.arange(h, device="cuda") // (h // kv)
    Q, K, V, dO = (None if f[x] is None else f[x].double() for x in ("q", "k", "v", "grad"))
    out, dQ, dK, dV = torch.zeros_like(Q), torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V)
    dT = None if f["table"] is None else torch.zeros(f["table"].shape, dtype=torch.float64, device="cuda")
    p_at = q_at = 0
    for np_, nq in zip(points, queries):
        pts = p[p_at:p_at + np_]
        order = _exact_order(pts.cpu().numpy())
        chosen = _exact_blocks(pts.cpu().numpy(), order, q[q_at:q_at + nq].cpu().numpy(), case["blocks"])
        block_of_point = torch.empty(np_, dtype=torch.long, device="cuda")
        block_of_point[torch.from_numpy(order).cuda()] = torch.arange(np_, device="cuda") // BLOCK
        chosen = torch.from_numpy(chosen).cuda()
        k, v = K[p_at:p_at + np_][:, group], V[p_at:p_at + np_][:, group]
        step = max(1, 60_000_000 // (h * np_))
        for at in range(q_at, q_at + nq, step):
            end = min(at + step, q_at + nq)
            hit = torch.zeros((end - at, (np_ + BLOCK - 1) // BLOCK + 1), dtype=torch.bool, device="cuda")
            hit.scatter_(1, chosen[at - q_at:end - q_at] % hit.shape[1], True)  # -1 is the spare last column
            seen = hit[:, block_of_point]
            logit = torch.einsum("mhc,nhc->hmn", Q[at:end], k) / math.sqrt(c)
            if dT is not None:
                d2 = torch.zeros((end - at, np_), device="cuda")
                for axis in range(p.shape[1]):
                    gap = q[at:end, axis, None] - pts[None, :, axis]
                    d2 = d2 + gap * gap
                bucket = torch.searchsorted(f["edges"], d2, right=True)
                logit = logit + f["table"].double()[:, bucket]
            weight = torch.softmax(logit.masked_fill(~seen, -math.inf), -1).nan_to_num(0)
            out[at:end] = torch.einsum("hmn,nhc->mhc", weight, v)
            if dO is None:
                continue
            slope = torch.einsum("mhc,nhc->hmn", dO[at:end], v)
            slope = weight * (slope - (weight * slope).sum(-1, keepdim=True))
            dQ[at:end] = torch.einsum("hmn,nhc->mhc", slope, k) / math.sqrt(c)
            dK[p_at:p_at + np_].index_add_(1, group, torch.einsum("hmn,mhc->nhc", slope, Q[at:end]) / math.sqrt(c))
            dV[p_at:p_at + np_].index_add_(1, group, torch.einsum("hmn,mhc->nhc", weight, dO[at:end]))
            if dT is not None:
                for head in range(h):
                    dT[head] += torch.bincount(bucket.reshape(-1), slope[head].reshape(-1), minlength=case["buckets"])
        p_at, q_at = p_at + np_, q_at + nq
    return [out] + ([dQ, dK, dV] if case["train"] else []) + ([dT] if case["train"] and dT is not None else [])


def _exact_bias(case, g):
    state = _bias_inputs(case, g)
    d2 = state["d2"] if case["per_head"] else state["d2"].unsqueeze(2).repeat(1, 1, case["heads"], 1)
    bucket = np.searchsorted(state["edges"].cpu().numpy(), d2.cpu().numpy(), side="right")
    table = state["table"].double().cpu().numpy()
    head = np.arange(case["heads"])[None, None, :, None]
    answer = [torch.from_numpy(table[head, bucket])]
    if case["train"]:
        at = (head * case["buckets"] + bucket).reshape(-1)
        total = np.bincount(at, state["grad"].double().cpu().numpy().reshape(-1), minlength=table.size)
        answer.append(torch.from_numpy(total.reshape(table.shape)))
    return answer


def exact(case, seed):
    """What ``run`` returns in 64 bits. Buckets and selections are whole numbers of float32
    distances by definition, and are taken from that arithmetic here too."""
    g = _generator(seed)
    if case["op"] == "bias":
        return _exact_bias(case, g)
    points, queries = _sizes(case)
    if case["op"] == "select":
        if sum(n * m for n, m in zip(points, queries)) // BLOCK > 150_000_000:
            return None
        p, q = _geometry(case, g)
        return [None, _exact_distances(case, p.cpu().numpy(), q.cpu().numpy())]
    if sum(n * m for n, m in zip(points, queries)) * case["heads"] > 5_000_000_000:
        return None
    return _exact_attend(case, g)
