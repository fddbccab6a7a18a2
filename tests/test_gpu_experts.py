"""Expert routing (csrc/tbe_experts.hip) against plain implementations in 64 bits.

Tolerances: a product or a sum in 32 bits is off by at most u = 2^-24 of its value, one in 64 by 2^-53, so a sum
of m products, in any order, by at most (m + 1) * u times the sum of the products' magnitudes; the one rounding
to the stored type by half a step, eps / 2 of the value, or half the step of the subnormals."""
import numpy as np
import pytest
import torch

from gpu_util import DEV

import table_batched_embeddings_experts as experts_mod
import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


def _unit(dtype):
    return 2.0 ** -53 if dtype == F64 else 2.0 ** -24


def assert_sum(got, want, magnitude, terms, dtype, what=""):
    """`want`: the exact value in 64 bits, `magnitude`: the sum of its terms' magnitudes."""
    got, want, magnitude = got.double().cpu(), want.double().cpu(), magnitude.double().cpu()
    info = torch.finfo(got.dtype if dtype is None else dtype)
    bound = (terms + 2) * _unit(dtype) * magnitude
    bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps / 2
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), "%s: %d of %d beyond the bound, worst %g over %g" % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float(bound[bad].min()))


def model_plan(ids, experts):
    flat = ids.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable")
    places = np.empty_like(order)
    places[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=experts + 1)[:experts])])
    return offsets, order, places.reshape(ids.shape), (key < experts).reshape(ids.shape)


def make_ids(seed, tokens, choices, experts, drop=0.0, dtype=np.int64, same=False):
    rs = np.random.RandomState(seed)
    ids = np.full((tokens, choices), experts - 1) if same else (rs.zipf(1.3, size=(tokens, choices)) - 1) % experts
    ids = np.where(rs.rand(tokens, choices) < drop, rs.choice([-1, experts, experts + 5, -2 ** 31], size=ids.shape), ids)
    return ids.astype(dtype)


PLANS = [(1, 1, 1, 0.0), (1, 2, 8, 0.0), (63, 1, 7, 0.1), (64, 1, 2, 0.0), (65, 3, 5, 0.5), (1000, 8, 255, 0.0),
         (1024, 8, 256, 0.2), (4096, 2, 1023, 0.0), (4097, 2, 64, 0.1), (700, 3, 1024, 0.0), (2048, 1, 4095, 0.3),
         (683, 3, 4095, 0.0), (50001, 5, 60, 0.17), (40000, 8, 300, 0.0), (30011, 4, 2000, 0.05), (300, 2, 9, 1.0),
         (9000, 1, 9, 1.0), (1024, 1, 255, 0.1), (1025, 1, 255, 0.1), (512, 2, 1023, 0.1), (513, 2, 1023, 0.0),
         (131072, 2, 200, 0.1), (131073, 2, 200, 0.1), (300001, 2, 100, 0.0), (65600, 8, 64, 0.1), (300000, 4, 3, 0.0),
         (5000, 3, 4000, 0.1), (2500, 1, 4095, 0.0), (20000, 2, 1023, 0.2)]


@pytest.mark.parametrize("tokens,choices,experts,drop", PLANS)
@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_plan_is_the_stable_sort(tokens, choices, experts, drop, dtype):
    ids = make_ids(tokens + experts, tokens, choices, experts, drop, dtype)
    print("plan", tokens, choices, experts, drop, flush=True)
    offsets, order, places = experts_mod.expert_plan(torch.from_numpy(ids).to(DEV), experts)
    want_offsets, want_order, want_places, _ = model_plan(ids, experts)
    assert np.array_equal(offsets.cpu().numpy(), want_offsets)
    assert np.array_equal(order.cpu().numpy(), want_order)
    assert np.array_equal(places.cpu().numpy(), want_places)


@pytest.mark.parametrize("tokens", [3, 20000])
def test_plan_of_one_popular_expert_and_of_far_ids(tokens):
    ids = make_ids(3, tokens, 2, 40, same=True)
    ids[::3, 0] = 2 ** 40 + 7       # whose low 32 bits are an expert's
    ids[1::3, 1] = -2 ** 63
    offsets, order, places = experts_mod.expert_plan(torch.from_numpy(ids).to(DEV), 40)
    want_offsets, want_order, want_places, _ = model_plan(ids, 40)
    assert np.array_equal(offsets.cpu().numpy(), want_offsets)
    assert np.array_equal(order.cpu().numpy(), want_order)
    assert np.array_equal(places.cpu().numpy(), want_places)


def test_plan_of_transposed_and_empty_ids():
    ids = make_ids(5, 3, 50, 11, 0.1).T  # [50, 3], strides of a transpose
    offsets, order, places = experts_mod.expert_plan(torch.from_numpy(ids.T.copy()).to(DEV).t(), 11)
    want = model_plan(np.ascontiguousarray(ids), 11)
    assert np.array_equal(offsets.cpu().numpy(), want[0]) and np.array_equal(places.cpu().numpy(), want[2])
    routing = ops.ExpertRouting(torch.empty(0, 4, dtype=torch.int32, device=DEV), 5)
    assert routing.expert_offsets.tolist() == [0] * 6 and routing.order.numel() == 0
    rows = routing.dispatch(torch.empty(0, 16, device=DEV))
    assert rows.shape == (0, 16)
    assert routing.combine(rows, torch.empty(0, 4, device=DEV)).shape == (0, 16)
    for experts in (1, 255, 1023, 1024, 4095):  # no token chose any of them
        none = ops.ExpertRouting(torch.empty(0, 2, dtype=torch.int64, device=DEV), experts)
        assert none.expert_offsets.numel() == experts + 1 and not none.expert_offsets.any()


# widths around the vector widths of every type, one vector more than a workgroup's, and strides
WIDTHS = [1, 2, 3, 5, 8, 33, 64, 100, 330, 1024, 2056, 8200]


def _problem(seed, tokens, choices, experts, D, dtype, drop, wdtype=None, misalign=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ids = make_ids(seed, tokens, choices, experts, drop)
    offsets, order, places, kept = model_plan(ids, experts)

    def values(n):
        # `misalign` elements into a wider buffer: another row distance and a base of no alignment
        flat = torch.randn(n, D + 2 * misalign, device=DEV, generator=gen, dtype=F32).to(dtype)
        return flat[:, misalign:misalign + D] if misalign else flat

    x, rows, grad = values(tokens), values(tokens * choices), values(tokens)
    weights = torch.rand(tokens, choices, device=DEV, generator=gen).to(wdtype or F32)
    routing = ops.ExpertRouting(torch.from_numpy(ids).to(DEV), experts)
    return dict(ids=ids, order=order, places=torch.from_numpy(places), kept=torch.from_numpy(kept), x=x, rows=rows,
                grad=grad, weights=weights, routing=routing, offsets=offsets)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32, F64])
@pytest.mark.parametrize("misalign", [0, 1])
def test_dispatch_moves_rows_bit_for_bit(D, dtype, misalign):
    tokens, choices, experts = (37, 3, 9) if D > 100 else (1201, 3, 60)
    p = _problem(D, tokens, choices, experts, D, dtype, 0.2, misalign=misalign)
    print("dispatch", D, dtype, misalign, flush=True)
    rows = p["routing"].dispatch(p["x"])
    kept = int(p["offsets"][-1])
    want = torch.zeros_like(rows)
    want[:kept] = p["x"][torch.from_numpy(p["order"][:kept] // choices).to(DEV)]
    assert torch.equal(rows, want)


def model_combine(p, rows, weights):
    """(value, sum of magnitudes) in 64 bits; dropped pairs are never read"""
    rows = rows.detach().double().cpu()
    picked = rows[p["places"].reshape(-1)].view(*p["places"].shape, -1)
    w = torch.ones_like(p["kept"], dtype=F64) if weights is None else weights.detach().double().cpu()
    terms = torch.where(p["kept"][..., None], picked * w[..., None], torch.zeros((), dtype=F64))
    return terms.sum(1), terms.abs().sum(1)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16), (F32, F32), (F64, F32),
                                          (F64, F64), (BF16, None)])
@pytest.mark.parametrize("misalign", [0, 1])
def test_combine_and_its_gradient(D, dtype, wdtype, misalign):
    tokens, experts = (37, 9) if D > 100 else (601, 60)
    choices = 1 + (D + (wdtype is None)) % 9  # 1 to 9
    p = _problem(D + 1, tokens, choices, experts, D, dtype, 0.3, wdtype, misalign)
    print("combine", D, dtype, wdtype, misalign, choices, flush=True)
    weights = None if wdtype is None else p["weights"]
    # what the dropped pairs hold is not looked at: their rows, their weights
    dropped = torch.where(p["kept"], torch.zeros((), dtype=torch.bool), torch.ones((), dtype=torch.bool))
    with torch.no_grad():
        p["rows"][p["places"][dropped].to(DEV)] = float("nan")
        if weights is not None:
            weights[dropped.to(DEV)] = float("inf")
    rows = p["rows"].detach().requires_grad_(True)
    if weights is not None:
        weights.requires_grad_(True)
    y = p["routing"].combine(rows, weights)
    want, magnitude = model_combine(p, rows, weights)
    assert_sum(y, want, magnitude, choices, dtype, "combine")

    inputs = (rows,) if weights is None else (rows, weights)
    grads = torch.autograd.grad(y, inputs, p["grad"])
    g = p["grad"].double().cpu()
    w = torch.ones(tokens, choices, dtype=F64) if weights is None else weights.detach().double().cpu()
    zero = torch.zeros((), dtype=F64)
    per_pair = torch.where(p["kept"][..., None], w[..., None] * g[:, None, :], zero)
    want_rows = torch.zeros(tokens * choices, D, dtype=F64)
    want_rows[p["places"].reshape(-1)] = per_pair.reshape(-1, D)
    assert_sum(grads[0], want_rows, want_rows.abs(), 0, dtype, "gradient of the rows")
    if weights is not None:
        picked = rows.detach().double().cpu()[p["places"].reshape(-1)].view(tokens, choices, D)
        terms = torch.where(p["kept"][..., None], picked * g[:, None, :], zero)
        # (the sum is made in the rows' accumulator, the rounding is to the weights' type)
        bound_type = F32 if dtype == F64 and wdtype == F32 else wdtype
        assert_sum(grads[1], terms.sum(2), terms.abs().sum(2), D, bound_type, "gradient of the weights")


@pytest.mark.parametrize("D", [3, 64, 330, 2056])
@pytest.mark.parametrize("dtype", [F16, BF16, F32, F64])
def test_dispatch_gradient_is_the_sum_of_a_tokens_rows(D, dtype):
    p = _problem(D + 2, 41, 5, 7, D, dtype, 0.4)
    x = p["x"].detach().requires_grad_(True)
    rows = p["routing"].dispatch(x)
    grad_rows = torch.randn(rows.shape, device=DEV).to(dtype)
    with torch.no_grad():  # what arrives for the zeros behind the last expert belongs to no token
        grad_rows[int(p["offsets"][-1]):] = float("nan")
    (gx,) = torch.autograd.grad(rows, x, grad_rows)
    want, magnitude = model_combine(p, grad_rows, None)
    assert_sum(gx, want, magnitude, 5, dtype, "gradient of the tokens")


def test_a_token_with_nothing_kept_is_zero_and_so_are_its_gradients():
    ids = torch.tensor([[-1, 4], [0, 1], [7, -3]], device=DEV)  # 4 experts: tokens 0 and 2 keep nothing
    routing = ops.ExpertRouting(ids, 4)
    assert routing.expert_offsets.tolist() == [0, 1, 2, 2, 2]
    x = torch.full((3, 20), 2.0, device=DEV, requires_grad=True)
    w = torch.full((3, 2), 0.5, device=DEV, requires_grad=True)
    y = routing.combine(routing.dispatch(x), w)
    assert y.tolist() == [[0.0] * 20, [2.0] * 20, [0.0] * 20]
    y.sum().backward()  # a broadcast gradient: both strides zero
    assert x.grad.tolist() == [[0.0] * 20, [1.0] * 20, [0.0] * 20]
    assert w.grad.tolist() == [[0.0, 0.0], [40.0, 40.0], [0.0, 0.0]]


def test_the_same_expert_twice_and_shared_weights():
    """A token may name an expert twice; weights may be one column, expanded."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, 3, (50, 1), device=DEV, generator=gen).expand(50, 4)
    routing = ops.ExpertRouting(ids, 3)
    x = torch.randn(50, 24, device=DEV, generator=gen, dtype=F64, requires_grad=True)
    w = torch.rand(50, 1, device=DEV, generator=gen, dtype=F64, requires_grad=True)
    g = torch.randn(50, 24, device=DEV, generator=gen, dtype=F64)
    y = routing.combine(routing.dispatch(x), w.expand(50, 4))
    gx, gw = torch.autograd.grad(y, (x, w), g)
    torch.testing.assert_close(y, 4 * w * x, rtol=1e-14, atol=1e-14)
    torch.testing.assert_close(gx, 4 * w * g, rtol=1e-14, atol=1e-14)
    torch.testing.assert_close(gw, 4 * (x * g).sum(1, keepdim=True), rtol=1e-13, atol=1e-13)


def test_only_the_gradients_that_are_wanted():
    """Frozen gates leave the rows unread, frozen rows get nothing written; the other gradient is the same."""
    p = _problem(12, 40, 3, 6, 72, BF16, 0.2)
    rows, weights = p["rows"].detach(), p["weights"].detach()
    both = [rows.clone().requires_grad_(True), weights.clone().requires_grad_(True)]
    want = torch.autograd.grad(p["routing"].combine(*both), both, p["grad"])
    (g,) = torch.autograd.grad(p["routing"].combine(both[0], weights), both[0], p["grad"])
    assert torch.equal(g, want[0])
    (g,) = torch.autograd.grad(p["routing"].combine(rows, both[1]), both[1], p["grad"])
    assert torch.equal(g, want[1])
    assert not p["routing"].combine(rows, weights).requires_grad
    with torch.no_grad():
        assert not p["routing"].combine(*both).requires_grad and not p["routing"].dispatch(p["x"]).requires_grad


def test_second_derivatives_are_refused():
    p = _problem(13, 10, 2, 4, 16, F32, 0.0)
    x = p["x"].detach().requires_grad_(True)
    rows = p["routing"].dispatch(x)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(rows, x, torch.ones_like(rows), create_graph=True)
    weights = p["weights"].requires_grad_(True)
    y = p["routing"].combine(rows.detach(), weights)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, weights, torch.ones_like(y), create_graph=True)


def test_rows_written_after_they_were_combined():
    p = _problem(14, 10, 2, 4, 16, F32, 0.0)
    rows, weights = p["rows"].clone(), p["weights"].requires_grad_(True)
    y = p["routing"].combine(rows, weights)
    rows.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_gradients_against_differences():
    ids = torch.from_numpy(make_ids(8, 7, 3, 5, 0.3)).to(DEV)
    routing = ops.ExpertRouting(ids, 5)
    x = torch.randn(7, 6, device=DEV, dtype=F64, requires_grad=True)
    w = torch.rand(7, 3, device=DEV, dtype=F64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x, w: routing.combine(torch.tanh(routing.dispatch(x)), w), (x, w))
    assert torch.autograd.gradcheck(lambda x: routing.combine(torch.tanh(routing.dispatch(x))), (x,))


def test_rows_beyond_32_bit_offsets():
    """n * k * D elements past 2^31: the far rows are the ones looked at."""
    tokens, choices, D = 33000, 2, 33000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    ids = torch.arange(tokens * choices, device=DEV).view(tokens, choices) % 5
    routing = ops.ExpertRouting(ids, 5)
    x = torch.arange(tokens, device=DEV, dtype=torch.int32).remainder(251).to(BF16)[:, None].expand(tokens, D).contiguous()
    rows = routing.dispatch(x)
    assert rows.numel() > 2 ** 31
    assert torch.equal(rows[:, 0], x[(routing.order // choices).long(), 0])
    assert torch.equal(rows[:, -1], rows[:, 0])
    w = torch.full((tokens, choices), 0.25, device=DEV)
    y = routing.combine(rows, w)
    assert torch.equal(y[:, -1], (x[:, 0].float() * 0.5).to(BF16)) and torch.equal(y[:, 0], y[:, -1])
    del x
    g = torch.ones(tokens, D, device=DEV, dtype=BF16)
    grad_rows, grad_weights = experts_mod.compiled().expert_combine_backward(g, rows, routing.places, routing.expert_offsets, w)
    assert bool((grad_rows[-3:] == 0.25).all()) and bool((grad_rows[:, -1] == 0.25).all())
    want = rows[routing.places.view(-1).long(), 0].double().view(tokens, choices) * D
    assert_sum(grad_weights, want, want.abs(), D, F32)


def test_places_out_of_range_are_left_alone():
    """A caller's own places: what lies outside the rows is a dropped pair's, in reading and in writing."""
    places = torch.tensor([[0, 99], [-5, 1]], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 50], dtype=torch.int32, device=DEV)  # claims more rows than there are
    rows = torch.arange(16, device=DEV, dtype=F32).view(4, 4)
    assert torch.equal(ops.expert_combine(rows, places, offsets), rows[:2])
    grad_rows, grad_w = experts_mod.compiled().expert_combine_backward(torch.ones(2, 4, device=DEV), rows, places, offsets,
                                                      torch.ones(2, 2, device=DEV))
    assert torch.equal(grad_rows[:2], torch.ones(2, 4, device=DEV))
    assert grad_w.tolist() == [[6.0, 0.0], [0.0, 22.0]]
    offsets = torch.tensor([0, -3], dtype=torch.int32, device=DEV)  # and less than none
    assert not ops.expert_combine(rows, places, offsets).any()
    assert not ops.expert_dispatch(rows[:2], places, offsets)[:2].any()


def _layer(x, ids, w, scale, experts):
    routing = ops.ExpertRouting(ids, experts)
    return routing.combine(routing.dispatch(x) * scale, w)


def test_another_stream_and_a_captured_step():
    """Forward and backward inside a graph, replayed on new inputs, against the eager step bit for bit."""
    tokens, choices, experts, D = 3000, 4, 20, 72
    gen = torch.Generator(device=DEV).manual_seed(6)

    def draw():
        ids = torch.randint(-1, experts, (tokens, choices), device=DEV, generator=gen)
        return (torch.randn(tokens, D, device=DEV, generator=gen).to(BF16), ids,
                torch.rand(tokens, choices, device=DEV, generator=gen),
                torch.randn(tokens, D, device=DEV, generator=gen).to(BF16))

    def step(x, ids, w, g):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = _layer(x, ids, w, 1.5, experts)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), g)

    buffers = draw()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*buffers)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, step(*buffers)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step(*buffers)
    for _ in range(4):
        fresh = draw()
        for b, f in zip(buffers, fresh):
            b.copy_(f)
        graph.replay()
        eager = step(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_refusals_on_the_device():
    ids = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    routing = ops.ExpertRouting(ids, 3)
    x = torch.zeros(4, 8, device=DEV)
    rows = routing.dispatch(x)
    for call, needle in [
            (lambda: ops.ExpertRouting(ids.float(), 3), "int32 or int64"),
            (lambda: ops.ExpertRouting(ids[0], 3), "choices"),
            (lambda: ops.ExpertRouting(ids, 0), "num_experts"),
            (lambda: ops.ExpertRouting(ids, 5000), "num_experts"),
            (lambda: routing.dispatch(x[:3]), "one row per row"),
            (lambda: routing.dispatch(x.int()), "float16"),
            (lambda: routing.dispatch(x[0]), "rows, D"),
            (lambda: routing.combine(rows[:5], None), "8 rows"),
            (lambda: routing.combine(rows, torch.zeros(4, 3, device=DEV)), "choices"),
            (lambda: routing.combine(rows, torch.zeros(4, 2, device=DEV, dtype=F16)), "dtype"),
            (lambda: routing.combine(rows, torch.zeros(4, 2)), "device"),
            (lambda: ops.expert_combine(rows, routing.places.long(), routing.expert_offsets), "int32"),
            (lambda: ops.expert_combine(rows, routing.places.t(), routing.expert_offsets), "contiguous"),
            (lambda: ops.expert_combine(rows, routing.places, routing.expert_offsets.cpu()), "device")]:
        with pytest.raises(RuntimeError, match=needle):
            call()


@pytest.mark.parametrize("fp16", [False, True])
def test_a_layer_on_top_of_embedding_bags(fp16):
    """Bags -> tokens -> experts -> back, with its backward through the fused table update."""
    T, E, D, B, experts, choices = 3, 200, 32, 64, 6, 2
    dtype = F16 if fp16 else F32
    rs = np.random.RandomState(4)
    bags = ops.TableBatchedEmbeddingBags(T, E, D, optimizer=ops.Optimizer.SGD, learning_rate=0.1, fp16=fp16).cuda()
    start = bags.embedding_weights.detach().double().cpu()
    lengths = rs.randint(0, 5, size=T * B)
    offs = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    idx = rs.randint(0, E, size=int(offs[-1])).astype(np.int32)
    out = bags(torch.from_numpy(idx).to(DEV), torch.from_numpy(offs).to(DEV))
    tokens = out.reshape(B * T, D)
    ids = make_ids(9, B * T, choices, experts, 0.1)
    routing = ops.ExpertRouting(torch.from_numpy(ids).to(DEV), experts)
    matrices = (torch.randn(experts, D, D, device=DEV) * 0.2).to(dtype).requires_grad_(True)
    gates = torch.rand(B * T, choices, device=DEV, requires_grad=True)
    bounds = routing.expert_offsets.tolist()
    rows = routing.dispatch(tokens)
    done = [torch.tanh(rows[bounds[e]:bounds[e + 1]] @ matrices[e]) for e in range(experts)]
    y = routing.combine(torch.cat(done + [rows[bounds[-1]:]]), gates)
    (y.float() ** 2).sum().backward()

    # the same in 64 bits on the CPU
    table = start.requires_grad_(True)
    m64, g64 = matrices.detach().double().cpu().requires_grad_(True), gates.detach().double().cpu().requires_grad_(True)
    bag = torch.repeat_interleave(torch.arange(T * B), torch.from_numpy(lengths))
    picked = table[torch.from_numpy(idx).long() + E * (bag // B)]
    pooled = torch.zeros(T * B, D, dtype=F64).index_add(0, bag, picked)
    x64 = pooled.view(T, B, D).transpose(0, 1).reshape(B * T, D)
    ids_t = torch.from_numpy(ids)
    kept = (ids_t >= 0) & (ids_t < experts)
    per_choice = [torch.tanh(torch.bmm(x64[:, None], m64[ids_t[:, j].clamp(0, experts - 1)])[:, 0]) for j in range(choices)]
    y64 = sum(torch.where(kept[:, j, None], g64[:, j, None] * per_choice[j], torch.zeros((), dtype=F64))
              for j in range(choices))
    (y64 ** 2).sum().backward()
    # chained roundings of the layer's stages (gather, product of 32 terms, tanh, combine, and back): some 16 half
    # steps of the stored type
    tol = 16 * torch.finfo(dtype).eps / 2

    def near(got, want, what):
        got, want = got.detach().double().cpu(), want.detach()
        assert float((got - want).norm()) <= tol * float(want.norm()), what

    near(y, y64, "output")
    near(matrices.grad, m64.grad, "experts' gradient")
    near(gates.grad, g64.grad, "gates' gradient")
    # the table moved by -lr * gradient, rounded to its type
    moved = bags.embedding_weights.detach().double().cpu() - start.detach()
    step_rounding = torch.finfo(dtype).eps / 2 * start.detach().abs().max() * np.sqrt(start.numel())
    assert float((moved + 0.1 * table.grad).norm()) <= tol * float(0.1 * table.grad.norm()) + float(step_rounding)


def test_forward_mode_derivatives_are_refused():
    ids = torch.tensor([[0, 1], [1, 0]], device=DEV)
    routing = ops.ExpertRouting(ids, 2)
    x, rows, gates = torch.ones(2, 8, device=DEV), torch.ones(4, 8, device=DEV), torch.ones(2, 2, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: routing.dispatch(dual(x)), lambda: routing.combine(dual(rows), gates),
                     lambda: routing.combine(rows, dual(gates))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
