"""prefill_attention's bound on the number of sequences, without a GPU."""

from __future__ import annotations

from test_prefill_cpu import FULL, call, lib  # noqa: F401


def test_numbers_of_sequences_near_2_to_31_are_refused(lib):  # noqa: F811
    for seqs in (0x7fffffff, 0x7fffffff - 100):
        assert call(lib, **dict(FULL, seqs=seqs, heads=1, kv=1)) == 2
        assert b"too many" in lib.pkv_last_error_string()
