"""The operators of expert routing and of gradient clipping: their measured cases, their plain form in
elementary torch operations, and the calls a user's program makes of the framework's own.

  route    tokens sorted by expert: the stable order of the (token, choice) pairs by expert, and the
           tokens' rows in that order                                   (serving, prompts)
  combine  the experts' rows back in token order, weighted and summed   (serving, prompts)
  train    both with their gradients: the routed part of one training step of a mixture-of-experts layer
  clip     the global norm of a list of gradients, and the gradients scaled down to a norm
  table    the norm of the exact gradient of a batch's embedding tables (one row per distinct index), and
           the batch's output gradient scaled down to a norm

A pair whose expert lies outside [0, experts) is dropped: it takes part in nothing, and its place is behind
the last expert's rows."""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6  # added to the norm, so that a gradient of zeros stays one


def listed():
    return [
        # one token of a decoding step, two experts of eight
        dict(name="route_token", kind="route", tokens=1, experts=8, choices=2, width=512, dtype="bf16", ids="int64",
             drop=0.0, skew=0.5),
        # a long prompt batch over many experts
        dict(name="route_prompts", kind="route", tokens=32768, experts=128, choices=8, width=2048, dtype="bf16",
             ids="int64", drop=0.0, skew=0.5),
        # a decoding step of eight requests
        dict(name="combine_step", kind="combine", tokens=8, experts=8, choices=2, width=512, dtype="bf16",
             weights="f32", drop=0.0, skew=0.5),
        # narrow fp32 rows, as the towers on top of embedding tables have them, some pairs over capacity
        dict(name="combine_narrow", kind="combine", tokens=20011, experts=60, choices=3, width=100, dtype="f32",
             weights="f32", drop=0.1, skew=1.0),
        # the long prompt batch's way back
        dict(name="combine_prompts", kind="combine", tokens=32768, experts=128, choices=8, width=2048, dtype="bf16",
             weights="f32", drop=0.0, skew=0.5),
        # a small training step over a padded batch: a sixth of the pairs are dropped; a width that no vector divides
        dict(name="train_padded", kind="train", tokens=5003, experts=16, choices=2, width=330, dtype="f16",
             weights="f32", ids="int32", drop=0.17, skew=1.0),
        # a large training step
        dict(name="train_large", kind="train", tokens=16384, experts=64, choices=4, width=4096, dtype="bf16",
             weights="bf16", ids="int64", drop=0.0, skew=0.5),
        # a few small tensors whose norm stays within the limit: nothing is scaled, in place
        dict(name="clip_within", kind="clip", tensors=11, numel=60001, dtype="f32", clipped=False),
        # the dense towers of a recommender, clipped
        dict(name="clip_towers", kind="clip", tensors=120, numel=12000000, dtype="f32", clipped=True),
        # a large model's gradients in 16 bits, clipped
        dict(name="clip_large", kind="clip", tensors=300, numel=600000000, dtype="bf16", clipped=True),
        # two small tables, every row a few times at most
        dict(name="table_small", kind="table", tables=2, rows=1000, width=32, batch=64, bag=4, alpha=0.0, dtype="f32",
             clipped=True),
        # the framework's training benchmark: 64 tables, 5.2 million skewed lookups
        dict(name="table_batch", kind="table", tables=64, rows=100000, width=128, batch=4096, bag=20, alpha=1.05,
             dtype="f32", clipped=True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "combine", "combine", "train", "clip", "clip", "table"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind in ("route", "combine", "train"):
        # no more than the largest listed ones move
        most = (1 << 29 if kind != "train" else 1 << 28) * 2 // SIZES[dtype]
        experts = _spread(rng, 2, 256)
        choices = rng.randint(1, min(8, experts))
        width = _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            width = max(16, width // 8 * 8)
        tokens = _spread(rng, 1, min(32768, max(1, most // (choices * width))))
        case = dict(kind=kind, tokens=tokens, experts=experts, choices=choices, width=width, dtype=dtype,
                    drop=rng.choice([0.0, round(rng.uniform(0.01, 0.4), 3)]), skew=round(rng.uniform(0.0, 1.5), 2))
        if kind != "combine":
            case["ids"] = rng.choice(["int32", "int64"])
        if kind != "route":
            case["weights"] = rng.choice(["f32", dtype])
        return case
    if kind == "clip":
        numel = _spread(rng, 100, 600000000 * 2 // SIZES[dtype])
        return dict(kind=kind, tensors=_spread(rng, 1, min(300, numel)), numel=numel, dtype=dtype,
                    clipped=rng.random() < 0.6)
    dtype = rng.choice(["f32", "f16"])
    tables, rows, width = _spread(rng, 1, 64), _spread(rng, 50, 100000), 4 * _spread(rng, 1, 64)
    bag = _spread(rng, 1, 40)
    batch = _spread(rng, 1, min(4096, max(1, (5242880 * 128 // max(width, 128)) // (tables * bag))))
    return dict(kind=kind, tables=tables, rows=rows, width=width, batch=batch, bag=bag,
                alpha=rng.choice([0.0, round(rng.uniform(1.02, 1.3), 2)]), dtype=dtype, clipped=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------ inputs
def _expert_ids(case, gen):
    """[tokens, choices]: every token's experts, all different, some experts more popular than others;
    `drop` of the pairs belong to no expert (padding, or over an expert's capacity)."""
    n, e, k = case["tokens"], case["experts"], case["choices"]
    popular = -case["skew"] * torch.log(torch.arange(1, e + 1, device="cuda", dtype=torch.float32))
    popular = popular[torch.randperm(e, device="cuda", generator=gen)]
    uniform = torch.rand(n, e, device="cuda", generator=gen).clamp_(1e-7, 1.0 - 1e-6)
    scores = popular - torch.log(-torch.log(uniform))
    ids = torch.topk(scores, k, dim=1).indices
    if case["drop"]:
        ids = torch.where(torch.rand(n, k, device="cuda", generator=gen) < case["drop"], torch.full_like(ids, -1), ids)
    return ids.to(torch.int32) if case.get("ids") == "int32" else ids


def _randn(shape, dtype, gen):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)


def _gates(case, gen):
    """[tokens, choices]: what the router gives the chosen experts, summing to one."""
    logits = torch.randn(case["tokens"], case["choices"], device="cuda", generator=gen)
    return torch.softmax(logits, dim=1).to(DTYPES[case["weights"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2654435761 % (1 << 62) + 17)
    state = dict(case=case)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind in ("route", "combine", "train"):
        n, k, width = case["tokens"], case["choices"], case["width"]
        state["ids"] = _expert_ids(case, gen)
        if kind != "combine":
            state["x"] = _randn((n, width), dtype, gen)
        if kind != "route":
            state["gates"] = _gates(case, gen)
        if kind == "combine":  # the plan was made on the way to the experts, whose outputs are here
            state["offsets"], _, state["places"] = _plain_plan(state["ids"], case["experts"])
            state["rows"] = _randn((n * k, width), dtype, gen)
        if kind == "train":
            state["grad"] = _randn((n, width), dtype, gen)
            state["x"].requires_grad_(True)
            state["gates"].requires_grad_(True)
        return state
    if kind == "clip":
        # one bucket, as a data-parallel step keeps its gradients, and a view of it for every parameter
        count, numel = case["tensors"], case["numel"]
        cuts = torch.rand(count - 1, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
        cuts = [0] + sorted((cuts ** 2 * numel).long().tolist()) + [numel]
        sizes = [b - a for a, b in zip(cuts, cuts[1:])]
        bucket = torch.empty(numel, device="cuda", dtype=dtype)
        bucket.normal_(generator=gen)
        bucket.mul_(0.01)
        state["bucket"] = bucket
        state["gradients"] = list(torch.split(bucket, sizes))
        # the norm is near 0.01 * sqrt(numel)
        state["max_norm"] = 0.01 * math.sqrt(numel) * (0.3 if case["clipped"] else 3.0)
        if case["clipped"]:  # out of place, so that every pass has gradients to scale
            state["out_bucket"] = torch.empty_like(bucket)
            state["out"] = list(torch.split(state["out_bucket"], sizes))
        return state
    tables, rows, batch, bag = case["tables"], case["rows"], case["batch"], case["bag"]
    n = tables * batch * bag
    # ragged bags with n lookups in all, empty ones among them
    cuts = torch.randint(0, n + 1, (tables * batch - 1,), device="cuda", generator=gen).sort().values
    ends = torch.tensor([0, n], device="cuda")
    state["offsets"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
    uniform = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64).clamp_min_(1e-12)
    if case["alpha"]:  # a power law over the rows, by its inverse distribution function
        power = 1.0 - case["alpha"]
        drawn = (1.0 + uniform * ((rows + 1.0) ** power - 1.0)) ** (1.0 / power) - 1.0
    else:
        drawn = uniform * rows
    indices = torch.floor(drawn).clamp_(0, rows - 1)
    state["indices"] = indices.to(torch.int32)
    state["table_offsets"] = (torch.arange(tables, device="cuda") * rows).to(torch.int32)
    state["weights"] = torch.zeros(tables * rows, case["width"], device="cuda", dtype=dtype)
    state["grad"] = _randn((batch, tables, case["width"]), dtype, gen).mul_(0.01)
    state["max_norm"] = 0.01 * math.sqrt(n * case["width"]) * (0.3 if case["clipped"] else 1000.0)
    return state


# -------------------------------------------------------------------------------------- plain form
def _plain_plan(ids, experts):
    """(first row of every expert and the number of rows in all, pairs in sorted order, place of every pair)"""
    n, k = ids.shape
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts)).long()
    order = torch.sort(key, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(n * k, device=ids.device)
    counts = torch.zeros(experts + 1, device=ids.device, dtype=torch.int64)
    counts.index_add_(0, key, torch.ones_like(key))
    offsets = torch.zeros(experts + 1, device=ids.device, dtype=torch.int64)
    offsets[1:] = torch.cumsum(counts[:experts], 0)
    return offsets.to(torch.int32), order.to(torch.int32), places.view(n, k).to(torch.int32)


def _plain_dispatch(x, offsets, order, choices):
    """Rows in sorted order; zeros behind the last expert's."""
    kept = torch.arange(order.numel(), device=x.device) < offsets[-1]
    rows = x[(order // choices).long()]
    return torch.where(kept[:, None], rows, torch.zeros((), device=x.device, dtype=x.dtype))


def _plain_gathered(rows, offsets, places):
    """[tokens, choices, width] in 32 bits, zeros for the dropped pairs; and which pairs are kept."""
    kept = places < offsets[-1]
    g = rows[places.reshape(-1).long()].float().view(*places.shape, -1)
    return torch.where(kept[..., None], g, torch.zeros((), device=rows.device)), kept


def _plain_combine(rows, offsets, places, gates):
    g, kept = _plain_gathered(rows, offsets, places)
    return (g * gates.float()[..., None]).sum(1).to(rows.dtype)


def _plain_train(state):
    x, gates, grad = state["x"].detach(), state["gates"].detach(), state["grad"]
    offsets, order, places = _plain_plan(state["ids"], state["case"]["experts"])
    rows = _plain_dispatch(x, offsets, order, places.shape[1])
    y = _plain_combine(rows, offsets, places, gates)
    g, kept = _plain_gathered(rows, offsets, places)
    grad_gates = (g * grad.float()[:, None, :]).sum(2).to(gates.dtype)
    # the gradient of the experts' rows, in their own type, then of the tokens
    back = (gates.float()[..., None] * grad.float()[:, None, :]).to(rows.dtype).float()
    back = torch.where(kept[..., None], back, torch.zeros((), device=x.device))
    return y, back.sum(1).to(x.dtype), grad_gates


def _plain_scale(norm, max_norm):
    return torch.clamp(max_norm / (norm + EPS), max=1.0)


def _plain_clip(state):
    # the tensors tile their bucket, so that their squares' sum is the bucket's
    bucket = state["bucket"]
    norm = torch.sqrt(bucket.float().square().sum(dtype=torch.float64)).float()
    out = state.get("out_bucket", bucket)
    out.copy_(bucket.float() * _plain_scale(norm, state["max_norm"]))
    return out, norm


def _plain_table(state):
    grad, case = state["grad"], state["case"]
    batch, tables, width = grad.shape
    offsets = state["offsets"].long()
    bags = torch.repeat_interleave(torch.arange(tables * batch, device=grad.device), offsets[1:] - offsets[:-1],
                                   output_size=state["indices"].numel())
    table = bags // batch
    keys = state["table_offsets"].long()[table] + state["indices"].long()
    by_bag = grad.float().transpose(0, 1).reshape(tables * batch, width)
    exact = torch.zeros(state["weights"].shape[0], width, device=grad.device)
    exact.index_add_(0, keys, by_bag[bags])
    norm = torch.sqrt(exact.square().sum(dtype=torch.float64)).float()
    return (grad.float() * _plain_scale(norm, state["max_norm"])).to(grad.dtype), norm


# --------------------------------------------------------------------------------- the framework's
def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-ads-baselines_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import table_batched_embeddings_ops as ops
    return ops


def _own(state):
    ops = _framework()
    case = state["case"]
    kind = case["kind"]
    if kind == "route":
        routing = ops.ExpertRouting(state["ids"], case["experts"])
        return routing.dispatch(state["x"]), routing.expert_offsets, routing.order, routing.places
    if kind == "combine":
        return ops.expert_combine(state["rows"], state["places"], state["offsets"], state["gates"])
    if kind == "train":
        routing = ops.ExpertRouting(state["ids"], case["experts"])
        y = routing.combine(routing.dispatch(state["x"]), state["gates"])
        return (y.detach(),) + torch.autograd.grad(y, (state["x"], state["gates"]), state["grad"])
    if kind == "clip":
        norm = ops.clip_gradients(state["gradients"], state["max_norm"], out=state.get("out"))
        return state.get("out_bucket", state["bucket"]), norm
    return ops.clip_table_gradient(state["grad"], state["weights"], state["table_offsets"], state["indices"],
                                   state["offsets"], state["max_norm"])


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "route":
        offsets, order, places = _plain_plan(state["ids"], state["case"]["experts"])
        return _plain_dispatch(state["x"], offsets, order, places.shape[1]), offsets, order, places
    if kind == "combine":
        return _plain_combine(state["rows"], state["offsets"], state["places"], state["gates"])
    if kind == "train":
        return _plain_train(state)
    if kind == "clip":
        return _plain_clip(state)
    return _plain_table(state)


# ------------------------------------------------------------------------------------------- floor
def work(case):
    """What a pass cannot do without, each operator's inputs read once and its outputs written once."""
    size = SIZES[case["dtype"]]
    kind = case["kind"]
    if kind in ("route", "combine", "train"):
        n, k, width, drop = case["tokens"], case["choices"], case["width"], case["drop"]
        tokens, pairs = n * width * size, n * k * width * size
        kept = pairs * (1.0 - drop)
        ids = n * k * (4 if case.get("ids") == "int32" else 8)
        plan = ids + 2 * 4 * n * k + 4 * (case["experts"] + 1)
        route = plan + tokens + pairs
        if kind == "route":
            return dict(bytes=int(route), flops=n * k)
        gates = n * k * SIZES[case["weights"]]
        combine = kept + tokens + gates + 4 * n * k
        if kind == "combine":
            return dict(bytes=int(combine), flops=int(2 * n * k * width * (1.0 - drop)))
        # combine's gradient: the output's read, the rows read, the rows' gradient written; dispatch's: read and summed
        back = tokens + kept + pairs + 2 * gates + 4 * n * k + kept + tokens + 4 * n * k
        return dict(bytes=int(route + combine + back), flops=int(6 * n * k * width * (1.0 - drop)))
    if kind == "clip":
        return dict(bytes=case["numel"] * size * (2 if case["clipped"] else 1), flops=(3 if case["clipped"] else 2) * case["numel"])
    n = case["tables"] * case["batch"] * case["bag"]
    grad = case["batch"] * case["tables"] * case["width"]
    return dict(bytes=2 * grad * size + 4 * n + 4 * (case["tables"] * case["batch"] + 1),
                flops=n * case["width"] + 3 * grad)


# --------------------------------------------------------------------------------- 64 bits, for its error
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":  # the rows are copied; whole numbers have no other value
        flat = s["ids"].reshape(-1).cpu().numpy().astype(np.int64)
        flat = np.where((flat < 0) | (flat >= case["experts"]), case["experts"], flat)
        order = np.lexsort((np.arange(flat.size), flat))
        rows = torch.zeros(flat.size, case["width"], device="cuda", dtype=torch.float64)
        kept = int((flat < case["experts"]).sum())
        rows[:kept] = s["x"].double()[torch.from_numpy(order[:kept] // case["choices"]).cuda()]
        return rows, None, None, None
    if kind in ("combine", "train"):
        n, k, width = case["tokens"], case["choices"], case["width"]
        gates = s["gates"].detach().double()
        valid = (s["ids"] >= 0) & (s["ids"] < case["experts"])
        if kind == "combine":
            y = torch.zeros(n, width, device="cuda", dtype=torch.float64)
            for j in range(k):
                picked = s["rows"].index_select(0, s["places"][:, j].long()).double()
                y.addcmul_(picked, torch.where(valid[:, j], gates[:, j], torch.zeros_like(gates[:, j]))[:, None])
            return y
        x, grad = s["x"].detach().double(), s["grad"].double()
        share = torch.where(valid, gates, torch.zeros_like(gates)).sum(1, keepdim=True)
        dots = (x * grad).sum(1, keepdim=True)
        return x * share, grad * share, torch.where(valid, dots.expand(-1, k), torch.zeros_like(gates))
    if kind == "clip":
        total = torch.zeros((), device="cuda", dtype=torch.float64)
        for piece in torch.split(s["bucket"], 1 << 26):
            p = piece.double()
            total += torch.dot(p, p)
        norm = total.sqrt()
        ratio = min(1.0, s["max_norm"] / (float(norm) + EPS))
        return s["bucket"].double() * ratio, norm
    batch, tables, width = s["grad"].shape
    rows = case["rows"]
    position = torch.arange(s["indices"].numel(), device="cuda")
    bag = torch.searchsorted(s["offsets"].long(), position, right=True) - 1
    total = 0.0
    for t in range(tables):  # table by table: 64-bit rows of all of them would be many gigabytes
        mine = slice(int(s["offsets"][t * batch]), int(s["offsets"][(t + 1) * batch]))
        summed = torch.zeros(rows, width, device="cuda", dtype=torch.float64)
        summed.index_add_(0, s["indices"][mine].long(), s["grad"][:, t].double()[bag[mine] - t * batch])
        total += float((summed * summed).sum())
    norm = math.sqrt(total)
    ratio = min(1.0, s["max_norm"] / (norm + EPS))
    return s["grad"].double() * ratio, torch.tensor(norm, device="cuda", dtype=torch.float64)
