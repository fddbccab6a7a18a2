"""Gradient norm and clipping (csrc/tbe_clip.hip) against plain implementations in 64 bits.

Tolerances: squares are exact products of values of at most 32 bits added up in 64, so the sum of n of them is off
by at most n * 2^-53 of its value and the norm by half of that; storing it as float32 adds 2^-24 of its value (the
square root and a float64 norm 2^-52 at most).  A scaled value carries the norm's error, the scale's rounding to
32 bits (2^-24) and the product's (2^-24), then half a step of its own type."""
import math

import numpy as np
import pytest
import torch

from conftest import make_problem
from gpu_util import DEV, dev

import table_batched_embeddings as ext
import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


def norm64(gradients):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in gradients))


def norm_error(norm, n):
    return n * 2.0 ** -53 + (2.0 ** -52 if norm.dtype == F64 else 2.0 ** -24)


def assert_norm(norm, want, n):
    assert norm.shape == ()
    assert abs(float(norm) - want) <= norm_error(norm, n) * want * 1.01, (float(norm), want)


def assert_scaled(got, before, scale, norm, n):
    want = before.double() * scale
    info = torch.finfo(got.dtype)
    rel = norm_error(norm, n) + 2 * (2.0 ** -53 if got.dtype == F64 else 2.0 ** -24)
    if info.bits == 16:
        rel += info.eps / 2
    bound = 1.01 * rel * want.abs() + info.smallest_normal * info.eps / 2
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), float((got.double() - want).abs()[bad].max())


def make_list(seed, sizes, dtype, misalign=0, scale=0.1):
    """Tensors inside one buffer with guard elements between them: (tensors, buffer)."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    buffer = torch.randn(sum(sizes) + (misalign + 1) * (len(sizes) + 1), device=DEV, generator=gen).mul_(scale).to(dtype)
    at, tensors = misalign, []
    for s in sizes:
        tensors.append(buffer[at:at + s])
        at += s + misalign + 1
    return tensors, buffer


SIZES = [[1], [7], [8, 0, 9], [1023, 1, 4096, 16385], [100003, 3, 64 * 1024 + 5], [17 + i % 300 for i in range(300)],
         [3000001], [1 + i % 5 for i in range(700)]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), s[0]))
@pytest.mark.parametrize("dtype", [F16, BF16, F32, F64])
@pytest.mark.parametrize("misalign", [0, 1, 2])
def test_norm_and_clip(sizes, dtype, misalign):
    tensors, buffer = make_list(len(sizes), sizes, dtype, misalign)
    n = sum(sizes)
    before, whole = [t.clone() for t in tensors], buffer.clone()
    print("clip", len(sizes), n, dtype, misalign, flush=True)
    want = norm64(before)
    norm = ops.gradient_norm(tensors)
    assert norm.dtype == (F64 if dtype == F64 else F32)
    assert_norm(norm, want, n)

    # into other tensors, at another alignment
    outs, out_buffer = make_list(1, sizes, dtype, (misalign + 1) % 3)
    out_whole = out_buffer.clone()
    max_norm = 0.37 * want
    scale = max_norm / (want + 1e-6)
    norm = ops.clip_gradients(tensors, max_norm, out=outs)
    assert_norm(norm, want, n)
    assert torch.equal(buffer, whole), "the gradients were written"
    for o, b in zip(outs, before):
        assert_scaled(o, b, scale, norm, n)
        o.copy_(torch.zeros_like(o))
    for o, t in zip(make_list(1, sizes, dtype, (misalign + 1) % 3)[0], outs):
        t.copy_(o)
    assert torch.equal(out_buffer, out_whole), "elements outside the outputs were written"

    # in place: within the limit nothing changes, beyond it only the tensors do
    assert_norm(ops.clip_gradients(tensors, 2 * want), want, n)
    assert torch.equal(buffer, whole)
    norm = ops.clip_gradients(tensors, max_norm)
    assert_norm(norm, want, n)
    for t, b in zip(tensors, before):
        assert_scaled(t, b, scale, norm, n)
        t.copy_(b)
    assert torch.equal(buffer, whole), "elements outside the gradients were written"

    # the same lists again: the same bits
    again, _ = make_list(1, sizes, dtype, misalign)
    first = ops.gradient_norm(again)
    assert all(torch.equal(ops.gradient_norm(again), first) for _ in range(3))


def test_lists_of_several_types_and_orders():
    gen = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    tensors = [r(33, 17).to(BF16), r(5, 6, 7).double(), r(40, 30).t(), r(9).to(F16), r(()), r(2, 8, 4, 4).to(
        memory_format=torch.channels_last), torch.empty(0, 3, device=DEV)]
    before = [t.clone() for t in tensors]
    want, n = norm64(before), sum(t.numel() for t in tensors)
    norm = ops.clip_gradients(tensors, 1.5)
    assert norm.dtype == F64
    assert_norm(norm, want, n)
    for t, b in zip(tensors, before):
        assert_scaled(t, b, 1.5 / (want + 1e-6), norm, n)


@pytest.mark.parametrize("dtype", [BF16, F32, F64])
def test_values_at_the_ends_of_the_types(dtype):
    big = torch.finfo(dtype).max / 4
    if dtype != F64:  # squares far beyond 32 bits
        g = torch.full((1000,), big, device=DEV, dtype=dtype)
        norm = ops.gradient_norm([g])
        want = big * math.sqrt(1000)
        if want < torch.finfo(F32).max:
            assert abs(float(norm) - want) <= 0.005 * want
        else:
            assert math.isinf(float(norm))
        g = torch.full((4,), big, device=DEV, dtype=dtype)
        want = 2 * float(g[0].double())
        norm = ops.clip_gradients([g], 1.0)
        assert_norm(norm, want, 4)
        assert torch.allclose(g.double(), torch.full_like(g, 0.5).double(), rtol=2 ** -7)
    tiny = torch.full((64,), 1e-30, device=DEV, dtype=dtype)
    norm = ops.clip_gradients([tiny], 1.0)
    assert float(norm) > 0 and bool((tiny == torch.tensor(1e-30, dtype=dtype)).all())
    zeros = torch.zeros(64, device=DEV, dtype=dtype)
    assert float(ops.clip_gradients([zeros], 0.0)) == 0.0 and not zeros.any()


def test_infinities_and_nan():
    def clip(values, max_norm):
        g = torch.tensor(values, device=DEV)
        norm = ops.clip_gradients([g], max_norm)
        return float(norm), g.tolist()

    norm, g = clip([1.0, float("inf"), -2.0], 1.0)
    assert math.isinf(norm) and g[0] == 0.0 and math.isnan(g[1]) and g[2] == 0.0
    norm, g = clip([1.0, float("nan")], 1.0)
    assert math.isnan(norm) and all(map(math.isnan, g))
    norm, g = clip([1.0, float("inf")], float("inf"))  # no limit
    assert math.isinf(norm) and g == [1.0, float("inf")]
    norm, g = clip([3.0, 4.0], 0.0)
    assert norm == 5.0 and g == [0.0, 0.0]


def test_more_elements_than_32_bits_count():
    n = (1 << 31) + 4099
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of device memory")
    g = torch.ones(n, device=DEV, dtype=BF16)
    g[-3:] = 64.0
    norm = ops.clip_gradients([g], 0.25 * math.sqrt(n))
    want = math.sqrt(n - 3 + 3 * 4096.0)
    assert_norm(norm, want, 1 << 20)
    scale = 0.25 * math.sqrt(n) / want
    assert abs(float(g[-1]) - 64 * scale) <= 64 * scale * 2.0 ** -8 and abs(float(g[0]) - scale) <= scale * 2.0 ** -8
    assert bool((g[:-3] == g[0]).all())


def test_refusals():
    g = torch.zeros(8, 8, device=DEV)
    for call, needle in [
            (lambda: ops.clip_gradients([g[:, :3]], 1.0), "gaps"),
            (lambda: ops.gradient_norm([g[0].expand(4, 8)]), "gaps"),
            (lambda: ops.gradient_norm([g, torch.zeros(3)]), "GPU tensors"),
            (lambda: ops.gradient_norm([g.int()]), "float16"),
            (lambda: ops.gradient_norm([g, 3.0]), "must be tensors"),
            (lambda: ops.gradient_norm(7), "a list of tensors"),
            (lambda: ops.clip_gradients([g, g], 1.0), "share memory"),
            (lambda: ops.clip_gradients([g, g[2]], 1.0), "share memory"),
            (lambda: ops.clip_gradients([g], -1.0), "max_norm"),
            (lambda: ops.clip_gradients([g], float("nan")), "max_norm"),
            (lambda: ops.clip_gradients([g], 1.0, out=[]), "one tensor per"),
            (lambda: ops.clip_gradients([g], 1.0, out=[g.t()]), "strides"),
            (lambda: ops.clip_gradients([g], 1.0, out=[g.half()]), "types")]:
        with pytest.raises((RuntimeError, TypeError), match=needle):
            call()
    assert float(ops.gradient_norm(t for t in (g, g))) == 0.0  # an iterator will do


def test_autograd_learns_that_a_gradient_was_scaled():
    x = torch.full((4,), 3.0, device=DEV, requires_grad=True)
    y = x.detach().clone().requires_grad_(True)
    w = torch.ones(4, device=DEV)
    out = (y * w).sum()  # saves w
    ops.clip_gradients([w], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward()


def test_two_streams_at_once():
    a, _ = make_list(5, [400000, 77], F32, 1)
    b, _ = make_list(6, [300000, 99], F32, 0)
    want = [norm64(a), norm64(b)]
    before = [[t.clone() for t in a], [t.clone() for t in b]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    norms = []
    for s, tensors in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            norms.append(ops.clip_gradients(tensors, 1.0))
    torch.cuda.synchronize()
    for norm, w, tensors, start in zip(norms, want, (a, b), before):
        assert_norm(norm, w, 400077)
        for t, s in zip(tensors, start):
            assert_scaled(t, s, 1.0 / (w + 1e-6), norm, 400077)


def test_captured_and_replayed():
    sizes = [5000, 33, 70001]
    tensors, buffer = make_list(8, sizes, F32, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_gradients([t.clone() for t in tensors], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = ops.clip_gradients(tensors, 2.0)
    for seed in range(4):
        _, fresh = make_list(20 + seed, sizes, F32, 1, scale=0.1 if seed % 2 else 1e-4)
        buffer.copy_(fresh)
        graph.replay()
        eager, eager_buffer = make_list(20 + seed, sizes, F32, 1, scale=0.1 if seed % 2 else 1e-4)
        eager_norm = ops.clip_gradients(eager, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, eager_norm)
        assert all(torch.equal(t, e) for t, e in zip(tensors, eager))


def test_clip_grad_norm_over_a_model_with_bags():
    bags = ops.TableBatchedEmbeddingBags(2, 50, 16, optimizer=ops.Optimizer.SGD, learning_rate=0.1).cuda()
    tower = torch.nn.Sequential(torch.nn.Linear(32, 24), torch.nn.Linear(24, 1)).to(DEV)
    p = make_problem(3, 2, 50, 16, 20, 6, np.float32)
    out = bags(dev(p["indices"]), dev(p["offsets"]))
    tower(out.reshape(20, 32)).square().sum().backward()
    parameters = list(bags.parameters()) + list(tower.parameters()) + [torch.nn.Parameter(torch.ones(3, device=DEV))]
    before = [q.grad.clone() for q in tower.parameters()]
    want = norm64(before)
    norm = ops.clip_grad_norm_(parameters, 0.1 * want)
    assert_norm(norm, want, 1000)
    for q, b in zip(tower.parameters(), before):
        assert_scaled(q.grad, b, 0.1 * want / (want + 1e-6), norm, 1000)
    tower[0].bias.grad[0] = float("nan")
    kept = [q.grad.clone() for q in tower.parameters()]
    with pytest.raises(RuntimeError, match="not finite"):
        ops.clip_grad_norm_(parameters, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(q.grad, k) or torch.isnan(k).any() for q, k in zip(tower.parameters(), kept))


# ------------------------------------------------------------------------------------- the tables
def table_norm64(p):
    """(norm of the exact gradient, bound of what 32-bit (64-bit for fp64) sums may be off by)"""
    T, B, D = p["T"], p["B"], p["D"]
    bag = np.repeat(np.arange(T * B), np.diff(p["offsets"]))
    keys = p["table_offsets"].astype(np.int64)[bag // B] + p["indices"]
    g = p["grad_output"].astype(np.float64).transpose(1, 0, 2).reshape(T * B, D)[bag]
    if p["per_sample_weights"] is not None:
        g = g * p["per_sample_weights"].astype(np.float64)[:, None]
    uniq, inverse, counts = np.unique(keys, return_inverse=True, return_counts=True)
    exact, magnitude = np.zeros((uniq.size, D)), np.zeros((uniq.size, D))
    np.add.at(exact, inverse, g)
    np.add.at(magnitude, inverse, np.abs(g))
    unit = 2.0 ** -53 if p["grad_output"].dtype == np.float64 else 2.0 ** -24
    error = (counts[:, None] + 2) * unit * magnitude
    norm = math.sqrt((exact ** 2).sum())
    return norm, math.sqrt((error ** 2).sum()) + norm * (1e-12 if unit < 1e-10 else 2.0 ** -23)


TABLES = [dict(T=1, E=9, D=8, B=1, L=1, ragged=False), dict(T=1, E=1, D=64, B=255, L=1, ragged=False),
          dict(T=1, E=1, D=32, B=257, L=3, ragged=False), dict(T=2, E=3, D=128, B=64, L=40),
          dict(T=3, E=1000, D=100, B=50, L=9), dict(T=5, E=400, D=12, B=64, L=20, zipf=1.3),
          dict(T=2, E=50, D=4, B=300, L=10, zipf=1.1), dict(T=4, E=2000, D=260, B=100, L=12, zipf=1.2),
          dict(T=2, E=30, D=1028, B=40, L=30), dict(T=1, E=5000, D=64, B=4096, L=20, zipf=1.05),
          dict(T=1, E=100, D=36, B=512, L=64, zipf=1.5), dict(T=3, E=20, D=2056, B=10, L=70),
          # rows of tens of thousands of lookups: segments of more than 64 tiles, alone, at both ends and side by side
          dict(T=1, E=1, D=64, B=700, L=60, ragged=False), dict(T=2, E=2, D=24, B=1024, L=60),
          dict(T=1, E=30, D=264, B=500, L=90, zipf=2.0)]


@pytest.mark.parametrize("shape", TABLES, ids=lambda s: "T%(T)d_E%(E)d_D%(D)d_B%(B)d_L%(L)d" % s)
@pytest.mark.parametrize("dtype,weighted", [(np.float32, False), (np.float16, True), (np.float64, False),
                                            (np.float32, True), (np.float16, False)])
def test_table_gradient_norm(shape, dtype, weighted):
    p = make_problem(31, dtype=dtype, weighted=weighted, **shape)
    print("table norm", shape, dtype, weighted, flush=True)
    want, bound = table_norm64(p)
    args = [dev(p[k]) for k in ("grad_output", "weights", "table_offsets", "indices", "offsets")]
    max_norm = 0.4 * want
    clipped, norm = ops.clip_table_gradient(*args, max_norm, dev(p["per_sample_weights"]))
    assert abs(float(norm) - want) <= bound, (float(norm), want, bound)
    # scaled by what the norm says (its own error is the bound's)
    scale = max_norm / (float(norm) + 1e-6)
    assert_scaled(clipped, args[0], min(1.0, scale), norm, 1)
    assert torch.equal(args[0], dev(p["grad_output"])) and torch.equal(args[1], dev(p["weights"]))
    again, norm_again = ops.clip_table_gradient(*args, max_norm, dev(p["per_sample_weights"]))
    assert torch.equal(norm, norm_again) and torch.equal(clipped, again)


def test_table_gradient_norm_of_an_empty_batch():
    w = torch.ones(8, 4, device=DEV)
    z = torch.zeros(3, dtype=torch.int32, device=DEV)
    go = torch.ones(2, 1, 4, device=DEV)
    clipped, norm = ops.clip_table_gradient(go, w, z[:1], z[:0], z, 1.0)
    assert float(norm) == 0.0 and torch.equal(clipped, go)


@pytest.mark.parametrize("optimizer,fp16,weighted,stochastic", [
    ("SGD", False, False, False), ("SGD", True, False, False), ("EXACT_ROWWISE_ADAGRAD", False, True, False),
    ("EXACT_ROWWISE_ADAGRAD", True, False, True), ("APPROX_ROWWISE_ADAGRAD", False, False, False),
    ("APPROX_ROWWISE_ADAGRAD", True, True, False)])
def test_module_clips_before_its_update(optimizer, fp16, weighted, stochastic):
    """A clipped backward is the unclipped one on the scaled gradient, bit for bit."""
    dtype = np.float16 if fp16 else np.float32
    p = make_problem(7, T=3, E=200, D=64, B=128, L=20, dtype=dtype, weighted=weighted, zipf=1.2)
    idx, off, psw = dev(p["indices"]), dev(p["offsets"]), dev(p["per_sample_weights"])
    go = dev(p["grad_output"])
    want, bound = table_norm64(p)

    def module():
        m = ops.TableBatchedEmbeddingBags(3, 200, 64, optimizer=ops.Optimizer[optimizer], learning_rate=0.1, eps=0.01,
                                          fp16=fp16, stochastic_rounding=stochastic).cuda()
        m.embedding_weights.data.copy_(dev(p["weights"]))
        return m

    results = []
    for factor in (0.3, 50.0):
        clipped_module, plain_module = module(), module()
        clip = clipped_module.clip_gradient(factor * want)
        assert clip.norm is None
        torch.manual_seed(11)
        clipped_module(idx, off, psw).backward(go)
        assert abs(float(clip.norm) - want) <= bound
        scaled, norm = ops.clip_table_gradient(go, plain_module.embedding_weights.data, plain_module.table_offsets, idx,
                                               off, factor * want, psw)
        assert torch.equal(norm, clip.norm) and torch.equal(scaled, go) == (factor > 1)
        torch.manual_seed(11)
        plain_module(idx, off, psw).backward(scaled)
        assert torch.equal(clipped_module.embedding_weights, plain_module.embedding_weights)
        assert torch.equal(clipped_module.optimizer_state, plain_module.optimizer_state)
        results.append(clipped_module.embedding_weights.detach().clone())
        # off again
        assert clipped_module.clip_gradient(None) is None
        clipped_module(idx, off, psw).backward(go)
        assert torch.equal(clip.norm, norm)
    assert not torch.equal(*results)


def test_module_clip_refusals():
    m = ops.TableBatchedEmbeddingBags(1, 20, 8, optimizer=ops.Optimizer.EXACT_ROWWISE_ADAGRAD, eps=0.1).cuda()
    m.clip_gradient(1.0)
    idx, off = torch.zeros(4, dtype=torch.int32, device=DEV), torch.arange(0, 5, dtype=torch.int32, device=DEV)
    psw = torch.ones(4, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="per-sample weights"):
        m(idx, off, psw)
    with torch.no_grad():  # no backward to come
        m(idx, off, psw)
    with pytest.raises(RuntimeError, match="max_norm"):
        m.clip_gradient(-2.0)
    cached = ops.TableBatchedEmbeddingBags(1, 200, 8, managed=ops.EmbeddingLocation.HOST_CACHED, cache_slots=64).cuda()
    with pytest.raises(RuntimeError, match="row cache"):
        cached.clip_gradient(1.0)


def test_captured_clipped_table_step():
    p = make_problem(17, T=3, E=300, D=32, B=64, L=15, dtype=np.float32, zipf=1.2)
    table_offsets, idx, off = dev(p["table_offsets"]), dev(p["indices"]), dev(p["offsets"])
    w, go = dev(p["weights"]), dev(p["grad_output"])
    import tbe_native
    step = lambda w, idx, go: tbe_native.compiled().backward_clipped(
        tbe_native.OPT_SGD, go, w, table_offsets, idx, off, None, None, 0.1, 0.0, False, 3.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w.clone(), idx, go)
    torch.cuda.synchronize()
    eager = w.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = step(w, idx, go)
    for _ in range(4):
        idx.copy_(torch.randint(0, 300, idx.shape, device=DEV, dtype=torch.int32))
        go.copy_(torch.randn_like(go))
        graph.replay()
        eager_norm = step(eager, idx.clone(), go.clone())
        torch.cuda.synchronize()
        assert torch.equal(norm, eager_norm) and torch.equal(w, eager)


def test_graphs_captured_on_one_stream_replayed_on_two():
    """The scratch memory of a call is its graph's own: two graphs captured on one stream may run at once."""
    p = make_problem(19, T=2, E=400, D=32, B=256, L=30, dtype=np.float32, zipf=1.3)
    table_offsets, off = dev(p["table_offsets"]), dev(p["offsets"])
    w = dev(p["weights"])
    inputs = [(dev(p["indices"]), dev(p["grad_output"])),
              (torch.randint_like(dev(p["indices"]), 0, 400), torch.randn_like(dev(p["grad_output"])))]
    lists = [make_list(40, [70000, 501], F32, 1)[0], make_list(41, [70000, 501], F32, 1)[0]]

    def step(i):
        idx, go = inputs[i]
        return ops.clip_table_gradient(go, w, table_offsets, idx, off, 2.0) + (
            ops.clip_gradients(lists[i], 1.0, out=[torch.empty_like(t) for t in lists[i]]),)

    eager = [step(0), step(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.synchronize()
    graphs, captured = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.append(step(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_whole_training_step_with_experts_and_clipping():
    """Bags that clip their tables' gradient, an expert layer on top, dense gradients clipped together: the step is the
    unclipped one with every gradient scaled by its own norm's factor."""
    T, E, D, B, experts, choices = 3, 150, 32, 64, 5, 2
    p = make_problem(23, T, E, D, B, 8, np.float32, zipf=1.3)
    ids = torch.randint(-1, experts, (B * T, choices), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    gen = torch.Generator(device=DEV).manual_seed(3)
    matrices0 = torch.randn(experts, D, D, device=DEV, generator=gen) * 0.2
    gates0 = torch.rand(B * T, choices, device=DEV, generator=gen)
    lr = 0.5

    def step(table_limit, dense_limit):
        bags = ops.TableBatchedEmbeddingBags(T, E, D, optimizer=ops.Optimizer.SGD, learning_rate=lr).cuda()
        bags.embedding_weights.data.copy_(dev(p["weights"]))
        clip = bags.clip_gradient(table_limit)
        matrices, gates = (torch.nn.Parameter(t.clone()) for t in (matrices0, gates0))
        routing = ops.ExpertRouting(ids, experts)
        rows = routing.dispatch(bags(dev(p["indices"]), dev(p["offsets"])).reshape(B * T, D))
        bounds = routing.expert_offsets.tolist()
        done = [torch.tanh(rows[bounds[e]:bounds[e + 1]] @ matrices[e]) for e in range(experts)]
        y = routing.combine(torch.cat(done + [rows[bounds[-1]:]]), gates)
        (100.0 * y).square().sum().backward()
        norm = ops.clip_grad_norm_(list(bags.parameters()) + [matrices, gates], dense_limit)
        moved = bags.embedding_weights.detach().double() - dev(p["weights"]).double()
        return moved, matrices.grad.double(), gates.grad.double(), float(norm), float(clip.norm)

    free = step(float("inf"), float("inf"))
    table_norm = float(free[0].norm()) / lr  # every row moved by -lr times its gradient, but for the weights' rounding
    assert abs(free[4] - table_norm) <= 1e-3 * table_norm
    assert abs(free[3] - float(torch.cat([free[1].flatten(), free[2].flatten()]).norm())) <= 1e-6 * free[3]
    table_limit, dense_limit = 0.25 * free[4], 0.4 * free[3]
    clipped = step(table_limit, dense_limit)
    assert clipped[3:] == free[3:]  # the same norms before scaling
    for got, want, scale in ((clipped[0], free[0], table_limit / (free[4] + 1e-6)),
                             (clipped[1], free[1], dense_limit / (free[3] + 1e-6)),
                             (clipped[2], free[2], dense_limit / (free[3] + 1e-6))):
        # three roundings of the scaled values, and for the table the rounding of both sides' weights
        weights = 2 * 2.0 ** -24 * 0.01 * math.sqrt(got.numel()) if got is clipped[0] else 0.0
        step_rounding = 2.0 ** -24 * (float(want.norm()) + float(got.norm()))
        assert float((got - scale * want).norm()) <= 4 * 2.0 ** -24 * float(got.norm()) + 2 * step_rounding + weights


@pytest.mark.parametrize("count,numel", [(321, 13), (2000, 700), (9000, 40)])
@pytest.mark.parametrize("in_place", [True, False])
def test_lists_of_thousands_of_tensors(count, numel, in_place):
    """More lists, and more partial sums, than the form without a launch for the norm takes."""
    gen = torch.Generator(device=DEV).manual_seed(count)
    flat = torch.randn(count * numel, device=DEV, generator=gen)
    want_norm = flat.double().norm()
    tensors = list(torch.split(flat.clone(), numel))
    out = None if in_place else list(torch.split(torch.full_like(flat, float("nan")), numel))
    norm = ops.clip_gradients(tensors, 2.0, out=out)
    assert abs(float(norm) - float(want_norm)) <= 2.0 ** -23 * float(want_norm)  # one rounding, and sums in 64 bits
    assert torch.equal(norm, ops.gradient_norm(list(torch.split(flat, numel))))
    want = flat.double() * (2.0 / (norm.double() + 1e-6))
    got = torch.cat(tensors if in_place else out).double()
    # the scale's rounding to 32 bits and the product's
    assert bool(((got - want).abs() <= 2.01 * 2.0 ** -24 * want.abs()).all())
