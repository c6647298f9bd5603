"""Performance cases of the products whose weights a row chooses: the router, the experts' products, the weighted sum of
the experts' rows, and low-rank adapters beside a shared projection.

Rows are encoder frames: 1 for each live stream, 126 for a clip of 10 s, 187 or 188 for a chunk of 15 s, some 52 000 for
an hour in chunks.  The widths are those of the network (1024, feed-forward 4096, joint 640, 1025 tokens + 5 durations).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D, FF, H, OUT = 1024, 4096, 640, 1030
HOUR = 280 * 187  # frames of an hour in 15 s chunks
SILU = 1


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one step of two dozen live streams: the router's latency
        dict(name="route_streams", kind="route", rows=24, experts=32, k=2, bf16=False, normalize=True, masked=False),
        # an hour of chunks, some experts switched off for some rows
        dict(name="route_hour", kind="route", rows=HOUR, experts=128, k=4, bf16=True, normalize=False, masked=True),
        # the up-projection of those streams: a few rows for each of some twenty experts, bound by the weights
        dict(name="experts_streams_up", kind="grouped", rows=24, k=2, groups=32, K=D, N=FF, gather=True, fp8=False, act=SILU, f32=False),
        # a serving batch of 32 clips of 10 s, two experts a frame, rows picked through the router's order
        dict(name="experts_clips_up", kind="grouped", rows=32 * 126, k=2, groups=16, K=D, N=FF, gather=True, fp8=False, act=SILU, f32=False),
        # an hour of chunks through the down-projection, rows already in the experts' order
        dict(name="experts_hour_down", kind="grouped", rows=HOUR, k=1, groups=32, K=FF, N=D, gather=False, fp8=False, act=0, f32=False),
        # one output layer for each language: 1025 tokens and 5 durations, logits in 32 bits
        dict(name="heads_by_language", kind="grouped", rows=2503, k=1, groups=11, K=H, N=OUT, gather=False, fp8=False, act=0, f32=True),
        # the e4m3 form of the up-projection on seventy chunks
        dict(name="experts_fp8_up", kind="grouped", rows=70 * 188, k=1, groups=16, K=D, N=FF, gather=True, fp8=True, act=SILU, f32=False),
        # the experts' rows of the live streams back to one row each
        dict(name="combine_streams", kind="combine", rows=24, k=2, cols=D, f32=True),
        # the same for an hour of chunks and four experts a frame
        dict(name="combine_hour", kind="combine", rows=HOUR, k=4, cols=D, f32=False),
        # one frame of each of 24 streams, each with a customer's adapter: latency, bound by the shared weights
        dict(name="adapters_streams", kind="adapter", rows=24, segments=24, adapters=64, rank=16, K=D, N=FF, act=SILU, f32=False),
        # seventy chunks of as many customers through a square projection that adds to the 32-bit residual stream
        dict(name="adapters_chunks", kind="adapter", rows=70 * 188, segments=70, adapters=70, rank=16, K=D, N=D, act=0, f32=True),
        # an hour of chunks of eight customers, rank 64
        dict(name="adapters_hour", kind="adapter", rows=HOUR, segments=280, adapters=8, rank=64, K=D, N=FF, act=SILU, f32=False),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "grouped", "grouped", "grouped", "combine", "adapter", "adapter", "adapter"])
    if kind == "route":
        experts = _between(rng, 4, 256)
        return dict(kind=kind, rows=_between(rng, 1, HOUR), experts=experts, k=rng.randint(1, min(8, experts)), bf16=rng.random() < 0.5,
                    normalize=rng.random() < 0.5, masked=rng.random() < 0.5)
    if kind == "combine":
        return dict(kind=kind, rows=_between(rng, 1, HOUR), k=rng.randint(1, 4), cols=rng.choice([D, H, 1016, 2 * D]) if rng.random() < 0.7 else rng.randint(8, 1200),
                    f32=rng.random() < 0.5)
    K, N = rng.choice([(D, FF), (FF, D), (D, D), (H, OUT), (D, H), (8 * rng.randint(8, 200), rng.randint(60, 1400))])
    # no more multiplications than the largest listed case
    most = HOUR * D * FF // (K * N)
    if kind == "grouped":
        k = rng.choice([1, 1, 2, 4])
        fp8 = K % 16 == 0 and rng.random() < 0.3
        return dict(kind=kind, rows=_between(rng, 1, min(HOUR, most) // k), k=k, groups=_between(rng, 4, 64), K=K, N=N, gather=k > 1 or rng.random() < 0.3,
                    fp8=fp8, act=rng.choice([0, SILU, 2]), f32=rng.random() < 0.3)
    segments = _between(rng, 1, 280)
    rows = max(segments, _between(rng, 1, min(HOUR, most) * 7 // 8))
    return dict(kind=kind, rows=rows, segments=segments, adapters=_between(rng, 1, 70), rank=rng.choice([8, 16, 16, 32, 64]), K=K, N=N,
                act=rng.choice([0, SILU, 2]), f32=rng.random() < 0.3)


# ----------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 31))
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _e4m3(x):
    """Rows in e4m3 and their scales."""
    scale = x.abs().amax(-1).clamp(min=1e-12) / 448.0
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _routed(g, rows, k, groups):
    """Experts of unequal popularity, one in eight unused: the row of each place and the experts' offsets."""
    pull = _randn(g, groups, std=0.7)
    if groups >= 8:
        pull[3::8] = -1e4
    chosen = (torch.randn(rows, groups, generator=g, device="cuda") + pull).topk(k, dim=1).indices.reshape(-1)
    order = chosen.sort(stable=True).indices
    sizes = torch.bincount(chosen, minlength=groups)
    offsets = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int()
    slots = torch.empty_like(order)
    slots[order] = torch.arange(rows * k, device="cuda")
    return (order // k).int(), slots.int().reshape(rows, k), offsets, int(sizes.max())


def prepare(case, seed):
    g = _generator(seed)
    kind, rows = case["kind"], case["rows"]
    state = dict(case)
    if kind == "route":
        e, k = case["experts"], case["k"]
        x = _randn(g, rows, e, std=1.5) + _randn(g, e, std=0.5)
        if case["masked"]:
            off = torch.rand(rows, e, generator=g, device="cuda") < 0.2
            off &= (torch.rand(rows, 1, generator=g, device="cuda") < 0.3)
            off |= (torch.rand(rows, 1, generator=g, device="cuda") < 0.01)  # a padded frame has no expert
            x = x.masked_fill(off, -math.inf)
        state["logits"] = x.to(torch.bfloat16 if case["bf16"] else torch.float32)
        i32 = dict(dtype=torch.int32, device="cuda")
        state.update(experts_out=torch.empty(rows, k, **i32), weights=torch.empty(rows, k, device="cuda"), offsets=torch.empty(e + 1, **i32),
                     order=torch.empty(rows * k, **i32), slots=torch.empty(rows, k, **i32))
        return state
    if kind == "combine":
        k, cols = case["k"], case["cols"]
        state["y"] = _randn(g, rows * k, cols, dtype=torch.bfloat16)
        w = torch.rand(rows, k, generator=g, device="cuda") + 0.05
        state["weights"] = w / w.sum(1, keepdim=True)
        slots = torch.randperm(rows * k, generator=g, device="cuda").int().reshape(rows, k)
        slots[torch.rand(rows, k, generator=g, device="cuda") < 0.02] = -1  # dropped
        state["slots"] = slots
        state["out"] = torch.empty(rows, cols, dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
        return state
    K, N = case["K"], case["N"]
    state["bias"] = None
    if kind == "grouped":
        k, n = case["k"], case["groups"]
        order, _, state["offsets"], state["most"] = _routed(g, rows, k, n)
        state["order"] = order if case["gather"] else None
        a = _randn(g, rows if case["gather"] else rows * k, K)
        w = torch.empty(n, N, K, dtype=torch.float8_e4m3fn if case["fp8"] else torch.bfloat16, device="cuda")
        scales = torch.empty(n, N, device="cuda")
        for e in range(n):
            we = _randn(g, N, K, std=K ** -0.5)
            if case["fp8"]:
                w[e], scales[e] = _e4m3(we)
            else:
                w[e] = we.bfloat16()
        state["w"], state["bias"] = w, _randn(g, n, N, std=0.1)
        state["row_scale"] = state["col_scale"] = None
        if case["fp8"]:
            state["a"], state["row_scale"] = _e4m3(a)
            state["col_scale"] = scales
        else:
            state["a"] = a.bfloat16()
        state["out"] = torch.empty(rows * k, N, dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
        return state
    n, r, s = case["adapters"], case["rank"], case["segments"]
    cuts = (torch.randperm(rows - 1, generator=g, device="cuda")[:s - 1] + 1).sort().values if s > 1 else torch.empty(0, dtype=torch.int64, device="cuda")
    who = torch.randint(n, (s,), generator=g, device="cuda")
    who[torch.rand(s, generator=g, device="cuda") < 0.1] = -1  # customers without an adapter
    state["who"] = who[torch.searchsorted(cuts, torch.arange(rows, device="cuda"), right=True)].int()
    state["a"] = _randn(g, rows, K, dtype=torch.bfloat16)
    state["w"] = _randn(g, N, K, std=K ** -0.5, dtype=torch.bfloat16)
    state["bias"] = _randn(g, N, std=0.1)
    state["down"] = _randn(g, n, r, K, std=K ** -0.5, dtype=torch.bfloat16)
    state["up"] = _randn(g, n, N, r, std=0.5 * r ** -0.5, dtype=torch.bfloat16)
    state["scale"] = torch.rand(n, generator=g, device="cuda") + 0.5
    state["out"] = torch.empty(rows, N, dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------------ plain forms
def _act(x, act):
    if act == SILU:
        return x / (1.0 + torch.exp(-x))
    return torch.clamp(x, min=0.0) if act == 2 else x


def _route(s):
    rows, e, k = s["rows"], s["experts"], s["k"]
    x = s["logits"].float()
    x = torch.where(x > -math.inf, x, torch.full_like(x, -math.inf)).clamp(max=torch.finfo(torch.float32).max)
    best, which = torch.sort(x, dim=1, descending=True, stable=True)
    top, which = best[:, :k], which[:, :k].int()
    fine = top > -math.inf
    m = best[:, :1]
    part = torch.where(fine, torch.exp(top - m), torch.zeros_like(top))
    whole = part if s["normalize"] else torch.where(x > -math.inf, torch.exp(x - m), torch.zeros_like(x))
    weights = torch.where(fine, part / whole.sum(1, keepdim=True), torch.zeros_like(part))
    experts = torch.where(fine, which, torch.full_like(which, -1))
    flat = torch.where(fine, which, torch.full_like(which, e)).reshape(-1)
    perm = torch.sort(flat, stable=True).indices
    offsets = torch.searchsorted(flat[perm], torch.arange(e + 1, device="cuda", dtype=torch.int32)).int()
    place = torch.arange(rows * k, device="cuda", dtype=torch.int32)
    inside = place < offsets[e]
    order = torch.where(inside, (perm // k).int(), torch.full_like(place, -1))
    slots = torch.empty_like(place).scatter_(0, perm, torch.where(inside, place, torch.full_like(place, -1)))
    return dict(experts=experts, weights=weights, offsets=offsets, order=order, slots=slots.reshape(rows, k))


def _grouped(s):
    a, w, offsets = s["a"].float(), s["w"].float(), s["offsets"].long()
    if s["row_scale"] is not None:
        a = a * s["row_scale"][:, None]
        w = w * s["col_scale"][:, :, None]
    rows = a if s["order"] is None else a[s["order"].long()]
    n = rows.shape[0]
    # the groups side by side, each as long as the longest, for one batched product
    place = offsets[:-1, None] + torch.arange(s["most"], device="cuda")
    padded = rows[place.clamp(max=n - 1)]
    y = torch.bmm(padded, w.transpose(1, 2))
    i = torch.arange(n, device="cuda")
    e = torch.searchsorted(offsets[1:], i, right=True)
    out = _act(y[e, i - offsets[e]] + s["bias"][e], s["act"])
    return dict(out=out if s["f32"] else out.bfloat16())


def _combine(s):
    slots = s["slots"].long()
    w = torch.where(slots >= 0, s["weights"], torch.zeros_like(s["weights"]))
    out = (s["y"][slots.clamp(min=0)].float() * w[:, :, None]).sum(1)
    return dict(out=out if s["f32"] else out.bfloat16())


def _adapter(s):
    a, n, r, rows = s["a"].float(), s["adapters"], s["rank"], s["rows"]
    who = s["who"].long()
    mine = torch.nn.functional.one_hot(who.clamp(min=0), n).float() * (who >= 0).float()[:, None] * s["scale"]
    # every adapter's down-projection of every row, all but the row's own put to zero
    low = (a @ s["down"].float().reshape(n * r, -1).T).reshape(rows, n, r) * mine[:, :, None]
    up = s["up"].float().permute(0, 2, 1).reshape(n * r, -1)
    out = _act(a @ s["w"].float().T + low.reshape(rows, n * r) @ up + s["bias"], s["act"])
    return dict(out=out if s["f32"] else out.bfloat16())


# ------------------------------------------------------------------------------------------------------ the framework
_kept = {}  # the context and the workspace that a user's program keeps


def _context():
    import scriptrs_b200 as sb

    if "ctx" not in _kept:
        _kept["ctx"] = sb.Context(0)
    return sb, _kept["ctx"]


def _work(size):
    """One workspace for all calls: they run one after the other on the context's stream."""
    if _kept.get("size", 0) < size:
        _kept["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        _kept["size"] = size
        torch.cuda.synchronize()
    return _kept["work"].data_ptr()


def _at(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    sb, ctx = _context()
    kind, rows = s["kind"], s["rows"]
    if kind == "route":
        size = sb.route_topk_workspace(rows, s["experts"], s["k"])
        sb.route_topk(ctx, _at(s["logits"]), _at(s["experts_out"]), _at(s["weights"]), _at(s["offsets"]), _at(s["order"]), _at(s["slots"]),
                      rows, s["experts"], s["k"], _work(size), size, bf16=s["bf16"], normalize=s["normalize"])
        return dict(experts=s["experts_out"], weights=s["weights"], offsets=s["offsets"], order=s["order"], slots=s["slots"])
    out = s["out"]
    mode = 1 if s["f32"] else 0
    if kind == "combine":
        sb.combine_rows(ctx, _at(s["y"]), _at(s["slots"]), _at(s["weights"]), _at(out), rows, s["k"], s["cols"], s["y"].shape[0], out_mode=mode)
    elif kind == "grouped":
        sb.grouped_gemm(ctx, _at(s["a"]), _at(s["w"]), _at(out), _at(s["offsets"]), s["groups"], out.shape[0], s["N"], s["K"],
                        d_rows=_at(s["order"]), a_rows=s["a"].shape[0], d_bias=_at(s["bias"]), act=s["act"], out_mode=mode, fp8=s["fp8"],
                        d_row_scale=_at(s["row_scale"]), d_col_scale=_at(s["col_scale"]))
    else:
        size = sb.adapter_gemm_workspace(rows, s["rank"])
        sb.adapter_gemm(ctx, _at(s["a"]), _at(s["w"]), _at(s["down"]), _at(s["up"]), _at(s["who"]), _at(out), s["adapters"], s["rank"],
                        rows, s["N"], s["K"], _work(size), size, d_scale=_at(s["scale"]), d_bias=_at(s["bias"]), act=s["act"], out_mode=mode)
    return dict(out=out)


def run(state):
    if own:
        return _own(state)
    return {"route": _route, "grouped": _grouped, "combine": _combine, "adapter": _adapter}[state["kind"]](state)


# --------------------------------------------------------------------------------------------- what cannot be avoided
def _met(n, draws):
    """How many of n are met at least once in so many even draws."""
    return n * (1.0 - (1.0 - 1.0 / n) ** draws)


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "route":
        e, k = case["experts"], case["k"]
        return {"bytes": rows * e * (2 if case["bf16"] else 4) + 16 * rows * k + 4 * (e + 1), "flops": 4 * rows * e}
    if kind == "combine":
        k, cols = case["k"], case["cols"]
        return {"bytes": rows * k * (2 * cols + 8) + rows * cols * (4 if case["f32"] else 2), "flops": 2 * rows * k * cols}
    K, N, ob = case["K"], case["N"], 4 if case["f32"] else 2
    if kind == "grouped":
        k, eb = case["k"], 1 if case["fp8"] else 2
        used = _met(case["groups"] * (7 / 8 if case["groups"] >= 8 else 1), rows * k)
        scales = (4 * rows + 4 * used * N) if case["fp8"] else 0
        a_rows = rows if case["gather"] else rows * k
        return {"bytes": a_rows * K * eb + used * (N * K * eb + 4 * N) + scales + rows * k * N * ob + (4 * rows * k if case["gather"] else 0),
                "flops": 2 * rows * k * N * K}
    r, share = case["rank"], 0.9
    used = _met(case["adapters"], case["segments"] * share)
    return {"bytes": rows * (2 * K + 4 + N * ob) + N * (2 * K + 4) + used * (2 * r * (K + N) + 4),
            "flops": 2 * rows * N * K + 2 * share * rows * r * (K + N)}


# ------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    kind, rows = case["kind"], case["rows"]
    if kind == "route":
        e, k = case["experts"], case["k"]
        x = s["logits"].double().cpu().numpy()
        ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
        top = np.take_along_axis(x, ids, 1)
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.exp(x - x.max(1, keepdims=True))
            chosen = np.take_along_axis(p, ids, 1)
            weights = chosen / (chosen if case["normalize"] else p).sum(1, keepdims=True)
        ids[np.isneginf(top)] = -1
        weights[np.isneginf(top)] = 0.0
        flat = ids.reshape(-1)
        taken = np.flatnonzero(flat >= 0)
        placed = taken[np.argsort(flat[taken], kind="stable")]
        offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[taken], minlength=e))])
        order, slots = np.full(rows * k, -1), np.full(rows * k, -1)
        order[:placed.size] = placed // k
        slots[placed] = np.arange(placed.size)
        i32 = lambda v: torch.from_numpy(np.ascontiguousarray(v, np.int32))  # noqa: E731
        return dict(experts=i32(ids), weights=torch.from_numpy(weights), offsets=i32(offsets), order=i32(order), slots=i32(slots.reshape(rows, k)))
    if kind == "combine":
        out = torch.zeros(rows, case["cols"], dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            at = s["slots"][:, j].long()
            here = at >= 0
            out[here] += s["weights"][here, j, None].double() * s["y"][at[here]].double()
        return dict(out=out)
    act = {0: lambda v: v, SILU: lambda v: v * torch.sigmoid(v), 2: torch.relu}[case["act"]]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    if kind == "grouped":
        at, a = s["offsets"].tolist(), s["a"].double()
        for e in range(case["groups"]):
            lo, hi = at[e], at[e + 1]
            which = slice(lo, hi) if s["order"] is None else s["order"][lo:hi].long()
            y = a[which] @ s["w"][e].double().T
            if case["fp8"]:
                y = y * s["row_scale"].double()[which, None] * s["col_scale"][e].double()
            out[lo:hi] = act(y + s["bias"][e].double())
        return dict(out=out)
    y = s["a"].double() @ s["w"].double().T + s["bias"].double()
    for n in range(case["adapters"]):
        here = s["who"] == n
        y[here] += s["scale"][n].double() * ((s["a"][here].double() @ s["down"][n].double().T) @ s["up"][n].double().T)
    return dict(out=act(y))
