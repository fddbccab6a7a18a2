"""Expert routing and clipping at sizes beyond the caches: the forms that stream their accesses, the second launch of a row
movement and the second round of a grid, against plain implementations in 64 bits.  (Tolerances: test_gpu_experts.py,
test_gpu_clip.py.)"""
import math

import numpy as np
import pytest
import torch

from conftest import make_problem
from gpu_util import DEV, dev

import table_batched_embeddings_experts as experts_mod
import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
MB = 1 << 20


def needs(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("needs %d GiB of device memory" % gib)


def assert_scaled(got, before, scale, norm, n):
    """norm: its own rounding and the 64-bit sums'; then the scale's and the product's to 32 bits, half a step of 16."""
    info = torch.finfo(got.dtype)
    rel = n * 2.0 ** -53 + (3 * 2.0 ** -53 if got.dtype == F64 else 3 * 2.0 ** -24) + 2.0 ** -52
    rel += info.eps / 2 if info.bits == 16 else 0.0
    for g, b in zip(torch.split(got, 1 << 25), torch.split(before, 1 << 25)):
        want = b.double() * scale
        bad = ~((g.double() - want).abs() <= 1.01 * rel * want.abs() + info.smallest_normal * info.eps / 2)
        assert not bad.any(), float((g.double() - want).abs()[bad].max())


def cut(buffer, sizes, gap):
    """Tensors of these sizes inside the buffer, `gap` elements before each and behind the last."""
    tensors, at = [], gap
    for s in sizes:
        tensors.append(buffer[at:at + s])
        at += s + gap
    assert at <= buffer.numel()
    return tensors


# bytes of a list around the limits of 32 and 256 MB, where stores into outputs of their own, and all accesses, are streamed
@pytest.mark.parametrize("dtype", [F16, BF16, F32, F64])
@pytest.mark.parametrize("megabytes", [24, 40, 200, 300])
@pytest.mark.parametrize("count", [5, 70, 400])
@pytest.mark.parametrize("in_place", [False, True])
def test_clipping_beyond_the_caches(dtype, megabytes, count, in_place):
    element = torch.finfo(dtype).bits // 8
    whole = megabytes * MB // element
    rs = np.random.RandomState(count)
    cuts = np.sort(rs.randint(0, whole, size=count - 1))
    sizes = np.diff(np.concatenate([[0], cuts, [whole]])).tolist()
    sizes[count // 2] += 3  # (odd sizes, whatever was drawn)
    print("clip", dtype, megabytes, count, in_place, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(count + megabytes)
    n = sum(sizes)
    buffer = torch.randn(n + (count + 1), device=DEV, generator=gen, dtype=F32).to(dtype)
    tensors = cut(buffer, sizes, 1)
    start = buffer.clone()
    befores = cut(start, sizes, 1)
    want = math.sqrt(sum(float(t.double().square().sum()) for t in befores))
    max_norm = 0.25 * want
    out = None
    if not in_place:
        out_buffer = torch.full((n + 2 * (count + 1),), 7.0, device=DEV, dtype=dtype)
        out = cut(out_buffer, sizes, 2)
    norm = ops.clip_gradients(tensors, max_norm, out=out)
    unit = 2.0 ** -52 if dtype == F64 else 2.0 ** -24
    # (the oracle's own sums, by tensor, in 64 bits)
    assert abs(float(norm) - want) <= (2 * n * 2.0 ** -53 + unit) * want
    assert torch.equal(norm, ops.gradient_norm(befores))
    scale = max_norm / (want + 1e-6)
    for o, b in zip(tensors if in_place else out, befores):
        assert_scaled(o, b, scale, norm, 2 * n)
        o.zero_()
        b.zero_()
    # what lies between the tensors is as it was
    if in_place:
        assert torch.equal(buffer, start)
    else:
        assert float(out_buffer.double().sum()) == 7.0 * 2 * (count + 1)


@pytest.mark.parametrize("dtype,B", [(np.float32, 1100), (np.float32, 9000), (np.float16, 2200)])
def test_table_gradients_beyond_the_caches(dtype, B):
    """36, 295 and 36 MB of output gradients, scaled into a copy."""
    p = make_problem(61, T=64, E=100, D=128, B=B, L=2, dtype=dtype)
    args = [dev(p[k]) for k in ("grad_output", "weights", "table_offsets", "indices", "offsets")]
    clipped, norm = ops.clip_table_gradient(*args, 1.0)
    scale = 1.0 / (float(norm) + 1e-6)
    assert scale < 1.0
    assert_scaled(clipped.view(-1), args[0].view(-1), scale, norm, 1)
    wide = torch.zeros(64 * 100, 128, device=DEV, dtype=F64)
    bag = torch.repeat_interleave(torch.arange(64 * B, device=DEV), (args[4][1:] - args[4][:-1]).long())
    keys = args[2].long()[bag // B] + args[3].long()
    wide.index_add_(0, keys, args[0].transpose(0, 1).reshape(64 * B, 128)[bag].double())
    counts = torch.bincount(keys, minlength=64 * 100).max().item()
    want = float(wide.norm())
    # 32-bit sums of up to `counts` rows, of magnitudes that add up to at most sqrt(counts) times the norm or so; one
    # rounding of the norm
    assert abs(float(norm) - want) <= (counts ** 1.5 * 2.0 ** -24 + 2.0 ** -23) * want


# rows that fill whole 128-byte lines and rows that do not, for every lane group of combine's gradient, beyond 256 MB
ROWS = [(BF16, 64, 2), (BF16, 128, 3), (F16, 256, 1), (BF16, 2048, 8), (F32, 1000, 4), (F64, 500, 2), (BF16, 2056, 4),
        (BF16, 2816, 2), (F16, 2824, 3),
        (F32, 4096, 2), (BF16, 36, 5), (F16, 330, 2)]


@pytest.mark.parametrize("dtype,D,choices", ROWS)
@pytest.mark.parametrize("wdtype", [F32, None])
def test_rows_beyond_the_caches(dtype, D, choices, wdtype):
    row_bytes = D * torch.finfo(dtype).bits // 8
    tokens = (300 * MB) // (row_bytes * choices) + 5
    experts = 37
    print("rows", dtype, D, choices, tokens, wdtype, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(D)
    ids = torch.randint(-3, experts, (tokens, choices), device=DEV, generator=gen)
    routing = ops.ExpertRouting(ids, experts)
    kept = ids >= 0
    flat = torch.where(kept, ids, torch.full_like(ids, experts)).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    assert torch.equal(routing.order.long(), order)
    num_kept = int(kept.sum())
    x = torch.randn(tokens, D, device=DEV, generator=gen, dtype=F32).to(dtype)
    rows = routing.dispatch(x)
    assert torch.equal(rows[:num_kept], x[order[:num_kept] // choices]) and not rows[num_kept:].any()

    rows = torch.randn(tokens * choices, D, device=DEV, generator=gen, dtype=F32).to(dtype)
    rows[num_kept:] = float("nan")
    weights = None if wdtype is None else torch.rand(tokens, choices, device=DEV, generator=gen)
    inputs = [rows.requires_grad_(True)] + ([] if weights is None else [weights.requires_grad_(True)])
    y = routing.combine(rows, weights)
    grad = torch.randn(tokens, D, device=DEV, generator=gen, dtype=F32).to(dtype)
    grads = torch.autograd.grad(y, inputs, grad)

    info, unit = torch.finfo(dtype), 2.0 ** -53 if dtype == F64 else 2.0 ** -24
    places = routing.places.long()
    w = torch.ones(tokens, choices, device=DEV, dtype=F64) if weights is None else weights.detach().double()
    zero = torch.zeros((), device=DEV, dtype=F64)

    def check(got, want, magnitude, terms, info):
        bound = (terms + 2) * unit * magnitude
        bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps / 2
        assert bool(((got.double() - want).abs() <= bound).all())

    step = max(1, (32 * MB) // (D * choices))
    for t in range(0, tokens, step):  # in pieces: 64-bit copies of all the rows would be gigabytes
        here = slice(t, t + step)
        k, at = kept[here], places[here]
        picked = rows.detach()[at.reshape(-1)].view(*at.shape, D).double()
        terms = torch.where(k[..., None], picked * w[here][..., None], zero)
        check(y.detach()[here], terms.sum(1), terms.abs().sum(1), choices, info)
        g = grad[here].double()[:, None, :]
        want = torch.where(k[..., None], w[here][..., None] * g, zero)
        check(grads[0][at.reshape(-1)].view(*at.shape, D), want, want.abs(), 0, info)
        if weights is not None:
            dots = torch.where(k[..., None], picked * g, zero)
            check(grads[1][here], dots.sum(2), dots.abs().sum(2), D, torch.finfo(F32))


def test_more_vectors_than_a_launch_numbers():
    """2^31 and some (token, vector) pairs: dispatch and combine take two launches, each over whole tokens."""
    needs(90)
    tokens, D = 131077, 131072 + 8  # 16385 vectors a row
    ids = torch.arange(tokens, device=DEV, dtype=torch.int32)[:, None].remainder_(7) - 1  # -1: a seventh is dropped
    routing = ops.ExpertRouting(ids, 6)
    kept = int(routing.expert_offsets[-1])
    line = torch.arange(D, device=DEV, dtype=torch.int32).remainder(199).to(BF16)
    rows = routing.dispatch(line[None, :].expand(tokens, D))
    for r in range(0, tokens, 4096):
        part = rows[r:r + 4096]
        inside = max(0, min(4096, kept - r))
        assert bool((part[:inside] == line).all()) and not part[inside:].any()
    far = [0, 1, 7, tokens // 2, tokens - 2, tokens - 1]
    marks = torch.tensor([3.0, 5.0, 9.0, 17.0, 33.0, 65.0], device=DEV, dtype=BF16)
    for t, m in zip(far, marks):
        rows[int(routing.places[t, 0])] = m
    w = torch.full((tokens, 1), 2.0, device=DEV)
    y = routing.combine(rows, w)
    dropped = (ids[:, 0] < 0)
    for t, m in zip(far, marks):
        assert bool((y[t] == (0.0 if dropped[t] else 2 * m)).all())
        y[t] = 0.0 if dropped[t] else 2 * line
    for t in range(0, tokens, 4096):
        want = torch.where(dropped[t:t + 4096, None], torch.zeros((), device=DEV, dtype=BF16), 2 * line)
        assert torch.equal(y[t:t + 4096], want)


# pairs beyond one round of the grid's 2^22 workgroups: a wavefront a pair (four a workgroup), and a workgroup a pair
@pytest.mark.parametrize("pairs,D", [((1 << 24) + 77, 264), ((1 << 22) + 77, 2840)])
def test_combines_gradient_beyond_one_round_of_the_grid(pairs, D):
    needs(60)
    choices = 2
    tokens = (pairs + 1) // 2
    ids = torch.arange(tokens * choices, device=DEV, dtype=torch.int32).view(tokens, choices).remainder_(5) - 1
    routing = ops.ExpertRouting(ids, 4)
    # small whole numbers: the dot products are exact in 32 bits
    grad = (torch.arange(tokens, device=DEV, dtype=torch.int32).remainder_(3) + 1).to(BF16)[:, None].expand(tokens, D)
    marks = torch.arange(tokens * choices, device=DEV, dtype=torch.int32).remainder_(13).to(BF16)
    rows = marks[:, None].expand(tokens * choices, D)
    w = torch.full((tokens, choices), 0.5, device=DEV)
    grad_rows, grad_w = experts_mod.compiled().expert_combine_backward(grad, rows, routing.places, routing.expert_offsets, w)
    kept = ids >= 0
    want_w = torch.where(kept, marks[routing.places.long()].float() * grad[:, :1].float() * D, torch.zeros((), device=DEV))
    assert torch.equal(grad_w, want_w)
    per_pair = torch.where(kept, 0.5 * grad[:, :1], torch.zeros((), device=DEV, dtype=BF16)).reshape(-1)
    want_rows = torch.empty_like(per_pair)
    want_rows[routing.places.view(-1).long()] = per_pair
    for r in range(0, tokens * choices, 1 << 20):
        assert bool((grad_rows[r:r + (1 << 20)] == want_rows[r:r + (1 << 20), None]).all())


def test_nothing_is_written_where_an_error_was_asked_for():
    """error_if_nonfinite: every gradient keeps its bits, the one that holds the NaN among them."""
    parameters = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (1000, 7, 40000)]
    for i, q in enumerate(parameters):
        q.grad = torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
    parameters[1].grad[3] = float("nan")
    bits = [q.grad.view(torch.int32).clone() for q in parameters]
    with pytest.raises(RuntimeError, match="not finite"):
        ops.clip_grad_norm_(parameters, 0.01, error_if_nonfinite=True)
    assert all(torch.equal(q.grad.view(torch.int32), b) for q, b in zip(parameters, bits))


def test_an_infinite_limit_scales_nothing_but_where_the_norm_is_no_number():
    inf, nan = float("inf"), float("nan")
    for values, want in [([1.0, -inf, 3.0], [1.0, -inf, 3.0]), ([1.0, 2.0], [1.0, 2.0]), ([1.0, nan, inf], [nan] * 3)]:
        for out in (None, torch.zeros(len(values), device=DEV)):
            g = torch.tensor(values, device=DEV)
            ops.clip_gradients([g], inf, out=None if out is None else [out])
            got = g if out is None else out
            torch.testing.assert_close(got.cpu(), torch.tensor(want), rtol=0, atol=0, equal_nan=True)
