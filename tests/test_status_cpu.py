"""CPU: every bit of the status word has a name in the header and in the front end, and a message."""
import os
import re

import pytest

from conftest import PKG, ROOT


def test_bits_have_names():
    from pie_b200 import _lib

    with open(os.path.join(ROOT, "include", "paged_attn_b200.h")) as f:
        header = {n: int(v) for n, v in re.findall(r"(PA_STATUS_\w+) = (\d+)", f.read())}
    with open(os.path.join(PKG, "csrc", "pa_types.h")) as f:
        device = {int(v) for v in re.findall(r"\bST_\w+ = (\d+)", f.read())}
    front = {n: v for n, v in vars(_lib).items() if n.startswith("PA_STATUS_")}
    assert header == front
    assert device == set(header.values())


def test_bits_have_messages():
    from pie_b200 import _lib, ops

    for name, v in vars(_lib).items():
        if name.startswith("PA_STATUS_"):
            with pytest.raises(IndexError, match=rf"x: device status {v:#x}: \w+"):
                ops._raise_status_value("x", v)
