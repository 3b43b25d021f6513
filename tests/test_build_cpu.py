"""The oracle's build step where the reference checkout is absent."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("made", [False, True])
def test_reference_build_is_skipped_without_a_checkout(tmp_path, made):
    from oracle import build_oracle
    d = tmp_path / "reference"
    if made:
        d.mkdir()  # an empty directory is no checkout either
    assert build_oracle.build_reference(str(d)) == []
