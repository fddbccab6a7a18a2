"""Clipped updates of fp16 tables whose scaled gradient fp16 does not hold: few bits or none are left of an element
below 2^-14, and what rounding does to equal elements adds up over a row's lookups.  The update then multiplies the
sums, in 32 bits."""
import math

import numpy as np
import pytest
import torch

from conftest import make_problem
from gpu_util import DEV, dev

import tbe_native
import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # a 32-bit rounding, relative
STEP = 2.0 ** -10  # of fp16; a rounding to nearest is off by half of it


def module(T, E, D, optimizer, lr, eps, weights, stochastic=False):
    m = ops.TableBatchedEmbeddingBags(T, E, D, optimizer=ops.Optimizer[optimizer], learning_rate=lr, eps=eps, fp16=True,
                                      stochastic_rounding=stochastic).cuda()
    m.embedding_weights.data.copy_(weights)
    return m


@pytest.mark.parametrize("max_norm", [1.0, 0.1])
@pytest.mark.parametrize("optimizer,weighted,stochastic", [("SGD", False, False), ("EXACT_ROWWISE_ADAGRAD", False, False),
                                                           ("EXACT_ROWWISE_ADAGRAD", True, False),
                                                           ("EXACT_ROWWISE_ADAGRAD", False, True)])
def test_a_hot_row_under_a_strong_clip(max_norm, optimizer, weighted, stochastic):
    """One row of 903301 lookups.  Every gradient is 2^-10, so that the sums of them are exact in 32 bits; scaled ones
    would be 1.4e-7 and 1.4e-8, where fp16 has steps of 6e-8."""
    B, L, D, lr, eps = 3001, 301, 64, 1.0, 0.01
    n = B * L
    idx = torch.full((n,), 2, dtype=torch.int32, device=DEV)
    off = torch.arange(0, n + 1, L, dtype=torch.int32, device=DEV)
    go = torch.full((B, 1, D), 2.0 ** -10, device=DEV, dtype=torch.float16)
    psw = torch.full((n,), 0.5, device=DEV, dtype=torch.float16) if weighted else None
    m = module(1, 4, D, optimizer, lr, eps, torch.zeros(4, D), stochastic)
    clip = m.clip_gradient(max_norm)
    m(idx, off, psw).backward(go)
    G = n * 2.0 ** -10 * (0.5 if weighted else 1.0)
    norm = G * math.sqrt(D)
    assert abs(float(clip.norm) - norm) <= 2 * U * norm
    scale = max_norm / (norm + 1e-6)
    moved = m.embedding_weights.detach().double().cpu()
    assert not moved[[0, 1, 3]].any()
    # the norm, the factor, the rate times the factor and its product with the sum: a rounding each
    error = 5 * U
    if optimizer == "SGD":
        want = -lr * scale * G
    else:
        state = (scale * norm) ** 2
        # 64 squares and their sum, the factor twice
        state_error = (D + 1 + 2 * error / U) * U
        got = m.optimizer_state.double().cpu()
        assert abs(float(got[2]) - state) <= 1.01 * state_error * state and not got[[0, 1, 3]].any()
        want = -lr / (math.sqrt(state) + eps) * scale * G
        error += state_error / 2 + 4 * U  # the root, its sum with eps, the quotient
    error += STEP if stochastic else STEP / 2
    assert bool(((moved[2] - want).abs() <= 1.01 * error * abs(want)).all()), (float(moved[2, 0]), want)


def test_per_sample_weights_make_the_rounding_larger():
    """Weights of 30 and a limit of 500: scaled elements of 2.3e-6, 38.7 steps of fp16, would move the norm by 0.8 %."""
    B, L, D, lr, eps, max_norm = 3001, 301, 64, 1.0, 0.01, 500.0
    n = B * L
    idx = torch.zeros(n, dtype=torch.int32, device=DEV)
    off = torch.arange(0, n + 1, L, dtype=torch.int32, device=DEV)
    go = torch.full((B, 1, D), 2.0 ** -10, device=DEV, dtype=torch.float16)
    m = module(1, 2, D, "EXACT_ROWWISE_ADAGRAD", lr, eps, torch.zeros(2, D))
    clip = m.clip_gradient(max_norm)
    m(idx, off, torch.full((n,), 30.0, device=DEV, dtype=torch.float16)).backward(go)
    G = n * 30.0 * 2.0 ** -10  # (whole multiples of 2^-9 below 2^24 of them: exact sums)
    norm = G * math.sqrt(D)
    assert abs(float(clip.norm) - norm) <= 2 * U * norm
    state = (max_norm / (norm + 1e-6) * norm) ** 2
    assert abs(float(m.optimizer_state[0]) - state) <= 1.01 * (D + 11) * U * state


@pytest.mark.parametrize("optimizer,weighted", [("SGD", False), ("EXACT_ROWWISE_ADAGRAD", False),
                                                ("EXACT_ROWWISE_ADAGRAD", True), ("APPROX_ROWWISE_ADAGRAD", False),
                                                ("APPROX_ROWWISE_ADAGRAD", True)])
@pytest.mark.parametrize("max_norm", [1e-5, 1e-7])
def test_rows_looked_up_once_under_a_strong_clip(optimizer, weighted, max_norm):
    """Scaled gradients of 4e-8 and 4e-10, which fp16 rounds to 6e-8 and to nothing."""
    rows, D, eps = 1000, 64, 1e-12
    lr = 1e6 if optimizer == "SGD" else 1.0
    idx = torch.randperm(rows, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.int32)
    off = torch.arange(rows + 1, dtype=torch.int32, device=DEV)
    go = torch.ones(rows, 1, D, device=DEV, dtype=torch.float16)
    psw = torch.full((rows,), 0.75, device=DEV, dtype=torch.float16) if weighted else None
    m = module(1, rows, D, optimizer, lr, eps, torch.zeros(rows, D))
    clip = m.clip_gradient(max_norm)
    m(idx, off, psw).backward(go)
    g = 0.75 if weighted else 1.0
    norm = g * math.sqrt(rows * D)
    assert abs(float(clip.norm) - norm) <= 2 * U * norm
    scale = max_norm / (norm + 1e-6)
    moved, error = m.embedding_weights.detach().double().cpu(), 6 * U  # (one more for the per-sample weight)
    if optimizer == "SGD":
        want = -lr * scale
    else:
        state = D * (g * scale) ** 2
        state_error = (D + 3 + 2 * error / U) * U
        assert bool(((m.optimizer_state.double().cpu() - state).abs() <= 1.01 * state_error * state).all())
        want = -lr / (math.sqrt(state) + eps) * g * scale
        error += state_error / 2 + 4 * U
    bound = 1.01 * (error + STEP / 2) * abs(want) + 2.0 ** -25
    assert bool(((moved - want).abs() <= bound).all()), (float(moved[0, 0]), want)


# rows of few, of tens, of hundreds and of thousands of lookups, in vectors of 8 and of 4 elements, and rows of more than
# a wavefront of vectors
SHAPES = [dict(T=1, E=5000, D=64, B=512, L=20), dict(T=3, E=300, D=128, B=128, L=40, zipf=1.3),
          dict(T=1, E=4, D=36, B=512, L=64), dict(T=2, E=40, D=256, B=200, L=60, zipf=1.2),
          dict(T=2, E=30, D=516, B=100, L=60, zipf=1.2), dict(T=2, E=60, D=1032, B=80, L=40, zipf=1.2)]
OPTIMIZERS = [("SGD", False, False), ("EXACT_ROWWISE_ADAGRAD", False, False), ("EXACT_ROWWISE_ADAGRAD", True, True),
              ("APPROX_ROWWISE_ADAGRAD", False, False), ("APPROX_ROWWISE_ADAGRAD", True, False),
              ("APPROX_ROWWISE_ADAGRAD", False, True), ("APPROX_ROWWISE_ADAGRAD", True, True)]


def small_gradient(p):
    """About 2^-10, of values that fp16 holds; 64 times as large it holds them too."""
    return (p["grad_output"].astype(np.float32) * np.float32(2.0 ** -10)).astype(np.float16)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "E%(E)d_D%(D)d_B%(B)d_L%(L)d" % s)
@pytest.mark.parametrize("optimizer,weighted,stochastic", OPTIMIZERS)
def test_the_factor_is_a_power_of_two(shape, optimizer, weighted, stochastic):
    """A clip by 2^-6 of a gradient 2^6 times as large is the unclipped update, bit for bit: every product with a power
    of two is exact."""
    p = make_problem(51, dtype=np.float16, weighted=weighted, **shape)
    T, E, D = shape["T"], shape["E"], shape["D"]
    idx, off, psw = dev(p["indices"]), dev(p["offsets"]), dev(p["per_sample_weights"])
    small = dev(small_gradient(p))
    large = small * 64
    assert torch.equal(large.float(), small.float() * 64)
    print("factor", shape, optimizer, weighted, stochastic, flush=True)

    def made():
        return module(T, E, D, optimizer, 0.5, 1e-4, dev(p["weights"]), stochastic)

    plain, clipped = made(), made()
    _, norm = ops.clip_table_gradient(large, plain.embedding_weights.data, plain.table_offsets, idx, off, 1.0, psw)
    max_norm = (float(norm) + 1e-6) / 64
    assert max_norm < p["n"] * math.sqrt(D) * 2.0 ** -14  # the update multiplies
    clip = clipped.clip_gradient(max_norm)
    torch.manual_seed(5)
    clipped(idx, off, psw).backward(large)
    torch.manual_seed(5)
    plain(idx, off, psw).backward(small)
    assert torch.equal(clip.norm, norm)
    assert not torch.equal(plain.embedding_weights, dev(p["weights"]))
    assert torch.equal(clipped.embedding_weights, plain.embedding_weights)
    assert torch.equal(clipped.optimizer_state, plain.optimizer_state)

    # within the limit (below that bound all the same): the unclipped update
    plain, clipped = made(), made()
    clip = clipped.clip_gradient(max_norm * 1.01)
    torch.manual_seed(5)
    clipped(idx, off, psw).backward(small)
    torch.manual_seed(5)
    plain(idx, off, psw).backward(small)
    assert torch.equal(clipped.embedding_weights, plain.embedding_weights)
    assert torch.equal(clipped.optimizer_state, plain.optimizer_state)


def test_norms_that_are_no_numbers():
    n, D = 4096, 8
    idx = torch.zeros(n, dtype=torch.int32, device=DEV)
    off = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    for bad in (float("nan"), float("inf")):
        go = torch.ones(n, 1, D, device=DEV, dtype=torch.float16)
        go[7, 0, 3] = bad
        m = module(1, 2, D, "SGD", 1.0, 0.0, torch.ones(2, D))
        m.clip_gradient(0.5)
        m(idx, off).backward(go)
        w = m.embedding_weights.detach().cpu()
        assert math.isnan(float(w[0, 3])) and bool((w[1] == 1.0).all())
        # a norm that is no number spreads, an infinite one makes finite gradients zero
        rest = w[0, [0, 1, 2, 4, 5, 6, 7]]
        assert bool(torch.isnan(rest).all()) if math.isnan(bad) else bool((rest == 1.0).all())
    m = module(1, 2, D, "SGD", 1.0, 0.0, torch.ones(2, D))
    m.clip_gradient(0.0)
    m(idx, off).backward(torch.ones(n, 1, D, device=DEV, dtype=torch.float16))
    assert bool((m.embedding_weights == 1.0).all())


@pytest.mark.parametrize("optimizer", [tbe_native.OPT_SGD, tbe_native.OPT_APPROX_ROWWISE_ADAGRAD])
def test_captured_and_replayed(optimizer):
    p = make_problem(53, T=2, E=300, D=32, B=256, L=40, dtype=np.float16, zipf=1.2)
    table_offsets, idx, off = dev(p["table_offsets"]), dev(p["indices"]), dev(p["offsets"])
    w, go = dev(p["weights"]), dev(small_gradient(p))
    state = torch.zeros(w.shape[0], device=DEV)

    def step(w, state, idx, go):
        return tbe_native.compiled().backward_clipped(optimizer, go, w, table_offsets, idx, off, None,
                                                      None if optimizer == tbe_native.OPT_SGD else state, 0.5, 1e-4, False,
                                                      0.01)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w.clone(), state.clone(), idx, go)
    torch.cuda.synchronize()
    eager, eager_state = w.clone(), state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = step(w, state, idx, go)
    gen = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(4):
        idx.copy_(torch.randint(0, 300, idx.shape, device=DEV, dtype=torch.int32, generator=gen))
        go.copy_(torch.randn(go.shape, device=DEV, generator=gen) * 2.0 ** -10)
        graph.replay()
        eager_norm = step(eager, eager_state, idx.clone(), go.clone())
        torch.cuda.synchronize()
        assert torch.equal(norm, eager_norm) and torch.equal(w, eager) and torch.equal(state, eager_state)
