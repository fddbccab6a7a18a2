"""CPU-side checks of expert routing: what the entry points refuse before they touch a device."""
import ctypes

import pytest
import torch

import table_batched_embeddings_ops as ops
import tbe_native

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
NULL = ctypes.c_void_p(0)


def _message(rc, code=1):
    assert rc == code
    return tbe_native.load().tbe_last_error().decode()


def test_plan_refusals():
    lib = tbe_native.load()
    plan = lambda ids=P, width=4, pairs=10, experts=4, ws=P, nbytes=1 << 20: lib.tbe_expert_plan(
        ids, width, pairs, experts, P, P, P, ws, nbytes, NULL)
    assert "4 or 8 bytes" in _message(plan(width=2))
    assert "num_pairs" in _message(plan(pairs=-1))
    assert "num_pairs" in _message(plan(pairs=2 ** 31 - 1))
    assert "num_experts" in _message(plan(experts=0))
    assert "num_experts" in _message(plan(experts=tbe_native.MAX_EXPERTS + 1))
    assert "null" in _message(plan(ids=NULL))
    assert "workspace" in _message(plan(pairs=100000, nbytes=16), code=2)
    assert "workspace" in _message(plan(ws=NULL, pairs=100000), code=2)


def test_plan_workspace_query():
    lib = tbe_native.load()
    size = lib.tbe_expert_plan_workspace_bytes
    assert size(-1, 4) == size(2 ** 31 - 1, 4) == size(4, 0) == size(4, tbe_native.MAX_EXPERTS + 1) == 0
    assert size(100000, 4) > 0
    # a workspace sized for a maximum serves every smaller batch
    for experts in (1, 60, 255, 256, 1023, 1024, 4095):
        sizes = [size(n, experts) for n in (0, 1, 1024, 1025, 8193, 16384, 16385, 65536, 65537, 100000, 262144, 262145,
                                              300000, 524288, 524289, 1 << 20, (1 << 31) - 2)]
        assert sizes == sorted(sizes)


@pytest.mark.parametrize("change,needle", [
    (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(tokens=-1), "num_tokens"), (dict(choices=0), "choices"),
    (dict(experts=0), "num_experts"), (dict(D=0), "D must be"), (dict(tokens=2 ** 30, choices=2), "out of range"),
    (dict(stride=-8), "stride"), (dict(base=ctypes.c_void_p(4097)), "misaligned"), (dict(base=NULL), "null")])
def test_row_movement_refusals(change, needle):
    lib = tbe_native.load()
    a = dict(base=P, stride=8, dtype=1, tokens=4, choices=2, experts=3, D=8)
    a.update(change)
    head = (a["base"], a["stride"], a["dtype"], a["tokens"], a["choices"], a["experts"], a["D"], P, P)
    assert needle in _message(lib.tbe_expert_dispatch(*head, P, NULL))
    assert needle in _message(lib.tbe_expert_combine(*head, P, 0, P, NULL))
    assert needle in _message(lib.tbe_expert_combine_backward(P, 8, *head, P, 0, P, P, NULL))


def test_weights_type_refusals():
    lib = tbe_native.load()
    assert "weights" in _message(lib.tbe_expert_combine(P, 8, 1, 4, 2, 3, 8, P, P, P, 3, P, NULL))
    assert "weights" in _message(lib.tbe_expert_combine_backward(P, 8, P, 8, 0, 4, 2, 3, 8, P, P, P, 2, P, P, NULL))


def test_embedding_entry_points_refuse_bfloat16():
    lib = tbe_native.load()
    assert "dtype" in _message(lib.tbe_forward(P, tbe_native.DTYPE_BF16, 4, P, 1, P, 4, P, 1, NULL, P, NULL))
    assert "dtype" in _message(lib.tbe_backward_sgd(P, P, tbe_native.DTYPE_BF16, 100, 0, 4, P, 1, P, 10, P, 1, 0.1, P,
                                                    1 << 30, NULL))


def test_cpu_tensors_are_rejected():
    ids = torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.ExpertRouting(ids, 3)
    places, offsets = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.expert_dispatch(torch.zeros(4, 8), places, offsets)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.expert_combine(torch.zeros(8, 8), places, offsets, torch.zeros(4, 2))
