"""CPU check of the same compiled kernels as tests/test_operator_resources.py: no
scalar register is kept in a vector register's lanes either (each use of one is then
a vector instruction more, in kernels that vector instructions bound)."""

from __future__ import annotations

import pytest

from tests.test_operator_resources import SOURCES, metadata


@pytest.mark.parametrize("src", SOURCES)
def test_no_scalar_spills(src):
    found = metadata(src)
    assert found
    spilled = {name: m["sgpr_spill_count"] for name, m in found.items() if m["sgpr_spill_count"]}
    assert not spilled, spilled
