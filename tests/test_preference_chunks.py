"""Chunks of the log-probabilities' backward, on the CPU."""
from __future__ import annotations

import pytest

from reversability_amd import _hip
from reversability_amd.preference import chunk_of, max_chunk


@pytest.mark.parametrize("padded", [64, 512, 50304])
@pytest.mark.parametrize("d", [8, 256, 4096, 8192, 65536])
def test_the_library_takes_every_chunk(padded, d):
    """The largest chunk of any width fits what one call takes."""
    rows = chunk_of(padded, d, None)
    assert 1 <= rows <= max_chunk(padded)
    assert _hip.library().rv_head_logp_bwd_workspace_bytes(rows, d, padded, padded) > 0


def test_a_callers_chunk_is_kept_where_it_can_be():
    assert chunk_of(64, 256, 100) == 100
    assert chunk_of(64, 8192, 1 << 22) < 1 << 22
