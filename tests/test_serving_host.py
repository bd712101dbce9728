"""CPU-only checks of what prompts and their samples pass through around the paged 8-bit cache: the entry points refuse bad arguments before anything reaches a GPU."""
import ctypes as C

import pytest

from test_paged_host import BAD, _error, _pages


def _rotate(**change):
    from kvquant._lib import Rotate, lib
    pages = change.pop("pages", None) or _pages()
    a = Rotate(C.pointer(pages), *[4096, 1024, 128, 1024] * 3, 4096, 4096, 4096, 4096, 0, 0, 0, 0, 0, 0, 2, 2, 8, 128, 0, 100)
    for name, value in change.items():
        setattr(a, name, value)
    return lib.odmkv_pages_write_rotated(C.byref(a), None)


@pytest.mark.parametrize("change,says", BAD, ids=[next(iter(c)) + "=" + str(next(iter(c.values()))) for c, _ in BAD])
def test_turning_into_a_bad_cache_is_refused(change, says):
    assert _rotate(pages=_pages(**change)) == -1 and says in _error(), _error()


def test_bad_turns_are_refused():
    from kvquant._lib import lib
    for change, says in ((dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(T=-1), "token count"), (dict(tokens=-1), "token count"), (dict(Hq=-1), "query heads"),
                         (dict(Hq=65536), "query heads"), (dict(turned=0), "dims to turn"), (dict(turned=136), "dims to turn"), (dict(turned=24), "dims to turn"), (dict(table=0), "table"),
                         (dict(positions=4096, starts=4096), "positions and starts"), (dict(q=0), "null"), (dict(q_out=0), "null"), (dict(k=0), "null"), (dict(v=0), "null"),
                         (dict(cosine=0), "null"), (dict(sine=0), "null"), (dict(q=4104), "aligned"), (dict(k_out=4100), "aligned"), (dict(sine=4100), "aligned"),
                         (dict(k_stride_t=100), "aligned"), (dict(q_stride_h=4), "aligned"), (dict(T=1 << 26), "too many")):
        assert _rotate(**change) == -1 and says in _error(), (change, _error())
    assert _rotate(T=0) == 0 and _rotate(offsets=4096, tokens=0) == 0                   # nothing to store
    assert lib.odmkv_pages_write_rotated(None, None) == -1 and "null" in _error()
