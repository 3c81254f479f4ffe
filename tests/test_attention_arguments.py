"""Sizes whose products pass 64 bits, refused by the attention entry points on the host."""
from __future__ import annotations

import pytest

from tests.test_kv_cache import _attention


@pytest.mark.parametrize("width", [1 << 31, (1 << 59) + 1, 1 << 60, (1 << 60) + 4, (1 << 63) - 1])
def test_a_table_wider_than_any(width):
    from vllm_webgpu_b200 import _lib as L
    assert _attention(table_width=width, table_row=width) == (L.ERR_SHAPE, L.ERR_SHAPE)
