"""evict_tokens refuses to write the new lengths over the old ones, which it still reads."""

from __future__ import annotations

from test_chunk_cpu import evict, lib  # noqa: F401  (lib: the fixture)


def test_refuses_lengths_in_place(lib):  # noqa: F811
    ptrs = [16] * 7
    assert evict(lib, ptrs) == 1 and b"seq_lens" in lib.pkv_last_error_string()
    assert evict(lib, [None] * 7, S=0) == 0
