"""How much one call of text_attention holds: what its launches cannot is refused before any of them, without a GPU."""

from __future__ import annotations

import pytest

from selas_amd import _lib

from .test_text_attention_checks import backward, forward, query

BACKWARD = "selas_text_attention_backward_workspace_bytes"


@pytest.mark.parametrize("kw", [dict(B=1 << 21, Lq=1, Lk=1), dict(B=1 << 20, Lq=2, Lk=1, H=8, Hk=8), dict(B=1 << 23, H=4, Hk=1, Lq=1, Lk=1)])
def test_more_few_row_items_than_a_grid_holds(kw):
    for call in (forward, query):
        with pytest.raises(_lib.Unsupported, match="2\\^32 threads"):
            call(**kw)
    assert query(**{**kw, "B": kw["B"] // 2 - 1}) == 0


@pytest.mark.parametrize("dtype", [_lib.BF16, _lib.F16])
def test_more_tiles_than_a_grid_holds(dtype):
    # One workgroup of 256 threads a head: 2^24 of them. fp16 also looks at every 64 rows of dO and v.
    kw = dict(B=1 << 22, Lq=1, Lk=1)
    with pytest.raises(_lib.Unsupported, match="2\\^32 threads"):
        query(BACKWARD, dtype=dtype, **kw)
    with pytest.raises(_lib.Unsupported, match="2\\^32 threads"):
        backward(dtype=dtype, ws=4096, size=1 << 60, **kw)
    assert query(BACKWARD, dtype=dtype, B=1 << 18, Lq=100, Lk=200) > 0
    more = dict(B=1 << 20, Lq=100, Lk=200)  # 2^22 workgroups of 128 queries, (2 + 4) x 2^22 of 64 rows
    if dtype == _lib.F16:
        with pytest.raises(_lib.Unsupported, match="2\\^32 threads"):
            query(BACKWARD, dtype=dtype, **more)
    else:
        assert query(BACKWARD, dtype=dtype, **more) > 0


def test_more_gradients_of_keys_than_a_grid_zeros():
    with pytest.raises(_lib.Unsupported, match="2\\^32 threads"):
        query(BACKWARD, B=1 << 13, Lq=0, Lk=1 << 13, Dh=64)
    assert query(BACKWARD, B=1 << 12, Lq=0, Lk=1 << 12, Dh=64) == 0


@pytest.mark.parametrize("kw", [dict(B=1 << 10, Lq=100, Lk=512), dict(Lq=1, Lk=1 << 27), dict(B=1, H=64, Hk=64, Lq=1 << 20, Lk=1 << 10)])
def test_large_calls_within_it_have_a_size(kw):
    assert query(**kw) >= 0 and query(BACKWARD, **kw) > 0 and query(BACKWARD, dtype=_lib.F16, **kw) > 0
