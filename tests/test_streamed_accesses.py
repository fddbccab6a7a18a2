"""The kernels that are chosen for data beyond the caches carry the streaming hint in every 16-byte access it is meant for:
the compiler may drop it without a word.  The device assembly of this repository's own sources is read."""
import os
import re
import subprocess

import pytest

import build


def vector_accesses(source, tmp_path):
    """{demangled kernel: [(is a store, has the hint) of every 16-byte access]}"""
    path = str(tmp_path / "kernels.s")
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.run([build._hipcc()] + flags + ["-S", "--cuda-device-only", os.path.join(build.CSRC, source), "-o", path],
                   check=True, stderr=subprocess.DEVNULL)
    kernels, current = {}, None
    with open(path) as lines:
        for line in lines:
            begin = re.match(r"(_Z\w+):", line)
            if begin:
                current = kernels.setdefault(begin.group(1), [])
            elif "Lfunc_end" in line:
                current = None
            elif current is not None:
                access = re.search(r"\b(?:global|flat|buffer)_(load|store)_dwordx4\b(.*)", line)
                if access:
                    current.append((access.group(1) == "store", re.search(r"\bnt\b", access.group(2)) is not None))
    return kernels


def flags_of(name, kernel):
    """The truth values among a kernel's template arguments, in order (None for another kernel)."""
    at = name.find(kernel + "I")
    return None if at < 0 else [v == "1" for v in re.findall(r"Lb([01])E", name[at:].split("EEv")[0] + "E")]


def test_scaled_gradients(tmp_path):
    kernels = vector_accesses("tbe_clip.hip", tmp_path)
    seen = 0
    for name, accesses in kernels.items():
        # (the list's own flag comes first)
        for kernel, loads, stores in (("12scale_kernel", 1, 2), ("19scale_joined_kernel", None, 1), ("17square_sum_kernel", 1, None)):
            flags = flags_of(name, kernel)
            if flags is None:
                continue
            seen += 1
            for is_store, hint in accesses:
                which = stores if is_store else loads
                assert hint == (flags[which] if which is not None else False), (name, is_store)
            assert any(not s for s, _ in accesses)
    assert seen >= 4 * (3 * 4 + 2 * 4 + 2 * 2)  # types; lists of two lengths, in place and not; what is streamed


def test_rows_of_experts(tmp_path):
    kernels = vector_accesses("tbe_experts.hip", tmp_path)
    seen = 0
    for name, accesses in kernels.items():
        flags = flags_of(name, "22expert_dispatch_kernel")
        if flags and flags[0]:
            seen += 1
            assert all(hint for is_store, hint in accesses if is_store) and any(s for s, _ in accesses)
        flags = flags_of(name, "21expert_combine_kernel")
        if flags and flags[0]:
            seen += 1
            assert all(hint for is_store, hint in accesses if not is_store) and any(not s for s, _ in accesses)
    assert seen == 1 + 7 * 3  # combine: seven pairs of types, three numbers of rows ahead
