"""CPU checks: results of paged_reserve and paged_truncate that lie over what other blocks still read are refused."""

from __future__ import annotations

import pytest

from test_capi_paged import CDX_EINVAL, _call, lib  # noqa: F401

B, ROWS = 4, 6
FREE = 1 << 20
RESERVE = "counts lengths positions B stride rows table table_ld width page free cap count starts new_counts " \
          "new_lengths new_positions new_count slots row_positions stream"
TRUNCATE = "to lengths positions B table table_ld width page free cap count new_lengths new_positions new_count stream"


def _reserve(lib):  # noqa: F811
    at = [FREE + 256 * i for i in range(13)]
    return _call(lib.cdx_paged_reserve, RESERVE, [at[0], at[1], at[2], B, 0, ROWS, at[3], 4, 4, 16, at[4], 9, *at[5:], None])


def _truncate(lib):  # noqa: F811
    at = [FREE + 256 * i for i in range(9)]
    return _call(lib.cdx_paged_truncate, TRUNCATE, [at[0], at[1], at[2], B, at[3], 4, 4, 16, at[4], 9, *at[5:], None])


def _cases(names, inputs, sizes):
    at = dict(zip([n for n in names.split() if n in inputs or n in sizes or n in ("table", "free")],
                  [FREE + 256 * i for i in range(13)]))
    for out, size in sizes.items():
        for x in inputs:
            n = 4 if x == "count" else 4 * B
            # The same place, the input's last word, and a result whose last word is the input's first.
            for where in (at[x], at[x] + n - 4, at[x] - size + 4):
                yield out, where


@pytest.mark.parametrize("out,where", _cases(RESERVE, ("counts", "lengths", "positions", "count"), {
    "starts": 4 * B, "new_counts": 4 * B, "new_lengths": 4 * B, "new_positions": 4 * B, "new_count": 4,
    "slots": 8 * ROWS, "row_positions": 4 * ROWS}))
def test_reserve_refuses_results_over_its_inputs(lib, out, where):  # noqa: F811
    assert _reserve(lib)(**{out: where}) == CDX_EINVAL
    assert b"memory of their own" in lib.cdx_last_error()


@pytest.mark.parametrize("out,where", _cases(TRUNCATE, ("to", "lengths", "positions", "count"), {
    "new_lengths": 4 * B, "new_positions": 4 * B, "new_count": 4}))
def test_truncate_refuses_results_over_its_inputs(lib, out, where):  # noqa: F811
    assert _truncate(lib)(**{out: where}) == CDX_EINVAL
    assert b"memory of their own" in lib.cdx_last_error()
