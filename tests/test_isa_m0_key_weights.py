"""The key weights' direct-to-LDS copies own M0, as those that tests/test_isa_m0.py checks
do: every M0 reference of key_weights_q8.hip's kernels is one of the copies' own."""
import os
import re

import pytest

import test_isa_m0 as base

SOURCE = "key_weights_q8.hip"


@pytest.mark.skipif(not os.path.exists(base.HIPCC), reason="hipcc is not installed")
def test_copies_own_m0(tmp_path, monkeypatch):
    monkeypatch.setitem(base.EXTRA, SOURCE, ["-mllvm", "-amdgpu-mfma-vgpr-form"])
    out = base.compile_isa(tmp_path, SOURCE)
    users, prev = 0, ""
    for text in base.instructions(out):
        assert not base.IMPLICIT.match(text), text
        if " lds" in text and text.startswith(("buffer_", "global_")):
            assert any(p.match(text) for p in base.ALLOWED), text
            assert not re.match(r"^s_(mov|add)_[bu]32 m0\b", prev), f"{prev} ; {text}"
        if re.search(r"\bm0\b", text):
            users += 1
            assert any(p.match(text) for p in base.ALLOWED), text
        prev = text
    assert users > 0
