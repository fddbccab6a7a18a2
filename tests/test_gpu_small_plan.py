"""Plans of small batches (one launch, in one workgroup) against numpy, bit for bit: gradient rows, the stable sort by
(table, row), segments and counters -- around the sizes where the form changes, and beyond it."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_util import DEV, dev

import tbe_native

pytestmark = pytest.mark.gpu

NUM_COUNTERS = 64 + 8 * 32  # integers from num_unique on that the update expects to be zero, but for the first


def plan(rows, lengths, indices, max_table_rows):
    """rows [T], lengths [T, B], indices [n] -> what the plan holds."""
    T, B = lengths.shape
    n = int(lengths.sum())
    table_offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(lengths.reshape(-1))]).astype(np.int32)
    lay = tbe_native.backward_workspace_layout(n, 4, tbe_native.DTYPE_F32, T)
    ws = torch.full((lay.total_bytes,), 0x5A, dtype=torch.uint8, device=DEV)
    to, idx, off = dev(table_offsets), dev(indices), dev(offsets)
    vp = lambda t: ctypes.c_void_p(t.data_ptr())
    tbe_native.check(tbe_native.load().tbe_plan_batch(
        vp(to), T, vp(idx), n, vp(off), B, int(table_offsets[-1]), max_table_rows, 4, tbe_native.DTYPE_F32, vp(ws),
        ws.numel(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    view = lambda o, c: ws[o:o + 4 * c].view(torch.int32).cpu().numpy()
    counters = view(lay.num_unique, NUM_COUNTERS)
    got = dict(grad_rows=view(lay.grad_rows, n), keys=view(lay.keys_sorted, n), positions=view(lay.positions_sorted, n),
               ids=view(lay.segment_ids, n), starts=view(lay.segment_starts, int(counters[0]) + 1))
    bags = np.repeat(np.arange(T * B), lengths.reshape(-1))
    keys = table_offsets[bags // B] + indices
    order = np.argsort(keys, kind="stable")
    sorted_keys = keys[order]
    heads = np.concatenate([[True], sorted_keys[1:] != sorted_keys[:-1]])
    want = dict(grad_rows=bags % B * T + bags // B, keys=sorted_keys, positions=order, ids=np.cumsum(heads) - 1,
                starts=np.concatenate([np.flatnonzero(heads), [n]]))
    for name in want:
        np.testing.assert_array_equal(got[name], want[name].astype(np.int32), err_msg=name)
    assert counters[0] == heads.sum() and not counters[1:].any()


def spread(rs, n, bags, empty):
    """n lookups over `bags` bags, about a share `empty` of them without any."""
    weights = np.where(rs.rand(bags) < empty, 0.0, rs.rand(bags))
    if weights.sum() == 0:
        weights[bags // 2] = 1.0
    return rs.multinomial(n, weights / weights.sum())


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 511, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097])
@pytest.mark.parametrize("T,B,E", [(1, 1, 1), (1, 33, 100000), (2, 64, 1000), (7, 19, 17), (64, 128, 100000),
                                   (1024, 8, 3), (3, 2731, 1 << 29)])
def test_small_plans(n, T, B, E):
    rs = np.random.RandomState(n + T)
    lengths = spread(rs, n, T * B, 0.5).reshape(T, B)
    indices = rs.randint(0, E, size=n).astype(np.int32)
    hot = rs.rand(n) < 0.3
    indices[hot] = E - 1
    rows = np.full(T, E)
    plan(rows, lengths, indices, 0)
    plan(rows, lengths, indices, E)


@pytest.mark.parametrize("n", [5, 1024, 3000])
def test_small_plans_of_ragged_tables(n):
    rs = np.random.RandomState(n)
    rows = np.array([3, 70000, 1, 513, 1 << 20, 1024])
    lengths = spread(rs, n, 6 * 50, 0.2).reshape(6, 50)
    lengths[2] = 0  # no lookup at all; one bag with all of a table's
    lengths[3, 1:], lengths[3, 0] = 0, 7
    table = np.repeat(np.arange(6), lengths.sum(1))
    indices = (rs.randint(0, 1 << 30, size=len(table)) % rows[table]).astype(np.int32)
    plan(rows, lengths, indices, int(rows.max()))


def test_bags_without_lookups_at_both_ends():
    lengths = np.zeros((4, 2048), int)
    lengths[1, 2047], lengths[2, 0], lengths[2, 5] = 100, 900, 24
    plan(np.full(4, 50), lengths, np.random.RandomState(1).randint(0, 50, size=1024).astype(np.int32), 50)
