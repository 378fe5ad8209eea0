"""Entries of the compiled kernels, and the status codes of kernels that lie in headers (no device)."""
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
