"""CPU-side checks of clipping's refusals, one call at a time with its own reason."""
import ctypes

import pytest

import tbe_native

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
NULL = ctypes.c_void_p(0)


def _calls(addresses, numels, dtypes, outputs=None, max_norm=1.0, norm=P, norm_dtype=0, ws=P, nbytes=1 << 20):
    lib = tbe_native.load()
    n = len(addresses)
    g, o = (ctypes.c_void_p * n)(*addresses), (ctypes.c_void_p * n)(*(outputs or addresses))
    counts, types = (ctypes.c_int64 * n)(*numels), (ctypes.c_int32 * n)(*dtypes)
    return dict(norm=lambda: lib.tbe_gradient_norm(g, counts, types, n, norm, norm_dtype, ws, nbytes, NULL),
                scale=lambda: lib.tbe_scale_gradients(g, o, counts, types, n, max_norm, norm, norm_dtype, NULL),
                clip=lambda: lib.tbe_clip_gradients(g, o, counts, types, n, max_norm, norm, norm_dtype, ws, nbytes, NULL))


def _reason(call):
    """(return code, message of this call)"""
    lib = tbe_native.load()
    assert lib.tbe_linearize(NULL, 0, NULL, 0, NULL, 0, NULL, NULL, NULL) != 0  # another message before it
    before = lib.tbe_last_error().decode()
    rc = call()
    message = lib.tbe_last_error().decode()
    assert rc != 0 and message != before
    return rc, message


@pytest.mark.parametrize("name", ["norm", "scale", "clip"])
@pytest.mark.parametrize("kwargs,needle", [
    (dict(dtypes=[4]), "dtype"), (dict(numels=[-1]), "element count"), (dict(numels=[(1 << 40) + 1]), "element count"),
    (dict(addresses=[0]), "null"), (dict(addresses=[4098]), "misaligned"), (dict(addresses=[1 << 48]), "address"),
    (dict(norm=NULL), "norm is null"), (dict(norm_dtype=1), "norm is F32 or F64")])
def test_every_list_call_gives_its_reason(name, kwargs, needle):
    a = dict(addresses=[4096], numels=[8], dtypes=[0])
    a.update(kwargs)
    rc, message = _reason(_calls(**a)[name])
    assert rc == 1 and needle in message


@pytest.mark.parametrize("name", ["scale", "clip"])
@pytest.mark.parametrize("kwargs,needle", [
    (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"), (dict(outputs=[4098]), "misaligned"),
    (dict(addresses=[4096, 4096], numels=[8, 8], dtypes=[0, 0]), "two outputs share"),
    (dict(addresses=[4096, 4096 + 28], numels=[8, 8], dtypes=[0, 0]), "two outputs share"),
    (dict(outputs=[4096 + 4]), "another tensor's gradient"),
    (dict(addresses=[4096, 8192], numels=[8, 8], dtypes=[0, 0], outputs=[12288, 12288]), "two outputs share"),
    (dict(addresses=[4096, 8192], numels=[8, 8], dtypes=[0, 0], outputs=[8192, 4096]), "another tensor's gradient"),
    (dict(addresses=[4096, 8192], numels=[8, 8], dtypes=[0, 0], outputs=[8208, 12288]), "another tensor's gradient"),
    (dict(addresses=[8192, 4096], numels=[8, 2048], dtypes=[0, 0], outputs=[16384, 8188]), "another tensor's gradient")])
def test_every_writing_call_gives_its_reason(name, kwargs, needle):
    a = dict(addresses=[4096], numels=[8], dtypes=[0])
    a.update(kwargs)
    rc, message = _reason(_calls(**a)[name])
    assert rc == 1 and needle in message


@pytest.mark.parametrize("name", ["norm", "clip"])
@pytest.mark.parametrize("kwargs", [dict(ws=NULL), dict(nbytes=0), dict(nbytes=64)])
def test_small_workspaces(name, kwargs):
    rc, message = _reason(_calls([4096], [8], [0], **kwargs)[name])
    assert rc == 2 and "workspace" in message


def test_scaling_needs_no_workspace_to_refuse_shared_memory():
    rc, message = _reason(_calls([4096, 4096], [8, 8], [0, 0], nbytes=0, ws=NULL)["scale"])
    assert rc == 1 and "two outputs share" in message
