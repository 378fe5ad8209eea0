"""Entries of the compiled kernels, and the status codes of kernels that lie in headers (no device)."""
import ctypes
import glob
import os
import re

import pytest
import torch

from bitnet_c_b200.csrc import build, ops

HERE = os.path.dirname(build.__file__)


def test_the_joining_form_of_decode_attention_has_no_entry_of_its_own():
    # it starts in front of its wait and relies on the kernel that bn_attention_shared launches ahead of it
    libraries = [build.library("attention_shared"), build.library("attention_decode_tc")]
    assert [hasattr(lib, "bn_attention_shared") for lib in libraries] == [True, False]
    assert [hasattr(lib, "bn_attention_decode_tc") for lib in libraries] == [False, True]
    assert not any(hasattr(lib, "bn_attention_decode_tc_join") for lib in libraries)


def _codes():
    for path in sorted(glob.glob(os.path.join(HERE, "*.cu*"))):
        with open(path) as f:
            for name, code in re.findall(r"#define (\w+_ERR_\w*WAIT) (\d+)", f.read()):
                yield os.path.splitext(os.path.basename(path))[0], name, int(code)


def test_codes_are_distinct_in_headers_too():
    codes = [code for *_, code in _codes()]
    assert sorted(codes) == list(range(1, len(codes) + 1)) and len(codes) >= 9


@pytest.mark.parametrize("family,name,code", list(_codes()))
def test_every_code_names_its_kernel(monkeypatch, family, name, code):
    cpu = torch.device("cpu")
    monkeypatch.setattr(ops, "_tc_status", {})
    monkeypatch.setattr(ops, "_scratch", {})
    monkeypatch.setattr(ops, "_SCRATCH_FLOATS", 1)
    ops.tc_status(cpu).fill_(code)
    with pytest.raises(ops.KernelError, match=rf"^{family}: "):
        ops.check_tc_status(cpu)


def test_sequences_without_anything_shared_are_refused_by_the_entry():
    # (it would launch nothing, and the sequences' results would be those of the call before)
    entry = build.library("attention_shared").bn_attention_shared
    entry.restype = ctypes.c_int
    p, i, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    at = p(1 << 12)  # (16-byte aligned; refused before anything is read)
    call = lambda n_seqs, n_items: entry(at, i(768), i(512), i(640), at, i(512), i(n_seqs), i(8), i(2), i(64), f(0.1), at, i(n_items), at, i(4), at, at, at, at, i(4),  # noqa: E731
                                         at, at, i(9), at, at, i(1), at, p(0))
    assert call(0, 0) == 0
    for n_items in (0, -1, 65536):
        assert call(3, n_items) == 1
