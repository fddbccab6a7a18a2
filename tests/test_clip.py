"""CPU-side checks of gradient norm and clipping: what the entry points refuse before they touch a device."""
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


def _list(addresses, numels, dtypes, outputs=None):
    n = len(addresses)
    return ((ctypes.c_void_p * n)(*addresses), (ctypes.c_void_p * n)(*(outputs or addresses)),
            (ctypes.c_int64 * n)(*numels), (ctypes.c_int32 * n)(*dtypes), n)


def _all(addresses, numels, dtypes, outputs=None, max_norm=1.0, norm=P, norm_dtype=0, ws=P, nbytes=1 << 20):
    lib = tbe_native.load()
    g, o, n, d, count = _list(addresses, numels, dtypes, outputs)
    return (lib.tbe_gradient_norm(g, n, d, count, norm, norm_dtype, ws, nbytes, NULL),
            lib.tbe_scale_gradients(g, o, n, d, count, max_norm, norm, norm_dtype, NULL),
            lib.tbe_clip_gradients(g, o, n, d, count, max_norm, norm, norm_dtype, ws, nbytes, NULL))


@pytest.mark.parametrize("kwargs,needle", [
    (dict(addresses=[4096], numels=[8], dtypes=[4]), "dtype"), (dict(addresses=[4096], numels=[-1], dtypes=[0]), "count"),
    (dict(addresses=[0], numels=[8], dtypes=[0]), "null"), (dict(addresses=[4098], numels=[8], dtypes=[0]), "misaligned"),
    (dict(addresses=[4096], numels=[8], dtypes=[0], norm=NULL), "norm"),
    (dict(addresses=[4096], numels=[8], dtypes=[0], norm_dtype=1), "norm")])
def test_list_refusals(kwargs, needle):
    for rc in _all(**kwargs):
        assert rc == 1
    assert needle in tbe_native.load().tbe_last_error().decode()


def test_clip_refusals():
    lib = tbe_native.load()
    for bad in (-1.0, float("nan")):
        _, scale, clip = _all([NULL.value or 0], [0], [0], max_norm=bad, nbytes=0)
        assert scale == 1 and clip == 1
        assert "max_norm" in lib.tbe_last_error().decode()
    norm, _, clip = _all([4096], [8], [0], nbytes=64, outputs=[0])
    assert norm == 2
    norm, scale, clip = _all([4096], [8], [0], ws=NULL, outputs=[4098])
    assert norm == 2 and scale == 1 and clip == 1
    assert lib.tbe_gradient_norm_workspace_bytes(-1) == 0
    sizes = [lib.tbe_gradient_norm_workspace_bytes(n) for n in (0, 1, 128, 129, 1000, 1 << 20)]
    assert sizes == sorted(sizes) and sizes[0] > 0


@pytest.mark.parametrize("addresses,outputs", [
    ([4096, 4096], None),                # the same tensor twice
    ([4096, 4096 + 28], None),           # the last element of one is the first of the other
    ([4096], [4096 + 4]),                # an output shifted against its gradient
    ([4096, 8192], [12288, 12288]),      # one output twice
    ([4096, 8192], [8192, 4096]),        # outputs swapped
    ([4096, 8192], [8192 + 16, 12288]),  # an output inside another tensor's gradient
])
def test_shared_memory_is_refused(addresses, outputs):
    _, scale, clip = _all(addresses, [8] * len(addresses), [0] * len(addresses), outputs, nbytes=0)
    assert scale == 1
    assert "share" in tbe_native.load().tbe_last_error().decode() or clip == 2
    _, scale, clip = _all(addresses, [8] * len(addresses), [0] * len(addresses), outputs)
    assert scale == clip == 1
    assert "share" in tbe_native.load().tbe_last_error().decode()


def test_table_norm_refusals():
    lib = tbe_native.load()
    call = lambda grad=P, dtype=0, D=8, T=1, B=1, n=10, ws=P, nbytes=1 << 30, norm=P, norm_dtype=0: \
        lib.tbe_table_gradient_norm(grad, dtype, D, T, B, n, NULL, ws, nbytes, norm, norm_dtype, NULL)
    for kwargs, needle in [(dict(grad=NULL), "null"), (dict(dtype=3), "dtype"), (dict(D=6), "multiple of 4"),
                           (dict(T=0), "positive"), (dict(n=-1), "num_indices"), (dict(norm=NULL), "norm"),
                           (dict(norm_dtype=1), "norm")]:
        assert needle in _message(call(**kwargs))
    assert "workspace" in _message(call(nbytes=16), code=2)
    assert "too wide" in _message(call(D=1 << 22, n=100000, nbytes=1 << 62), code=4)


def test_python_refusals():
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ops.gradient_norm([torch.zeros(4)])
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ops.clip_gradients([torch.zeros(4)], 1.0)
    with pytest.raises(RuntimeError, match="at least one"):
        ops.clip_gradients([], 1.0)
    p = torch.nn.Parameter(torch.zeros(4))
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0  # no gradient yet
    with pytest.raises(RuntimeError, match="2-norm"):
        ops.clip_grad_norm_([p], 1.0, norm_type=1.0)
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1), (4,))
    with pytest.raises(RuntimeError, match="dense gradients"):
        ops.clip_grad_norm_(p, 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.TableGradientClip(-1.0)
