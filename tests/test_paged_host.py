"""CPU-only checks of the paged 8-bit cache: its entry points refuse bad arguments before anything reaches a GPU, and the plain statement that the GPU tests
compare with does what it says."""
import ctypes as C

import pytest
import torch

import paged_rows as plain


def _pages(**change):
    from kvquant._lib import Pages
    p = Pages(2, 3, 4, 10, 5, 0, 0, *[4096] * 12)
    for name, value in change.items():
        setattr(p, name, value)
    return p


BAD = [(dict(rows=0), "shape"), (dict(rows=1025), "shape"), (dict(pages=0), "shape"), (dict(pages=1 << 24), "shape"), (dict(blocks=0), "shape"),
       (dict(Hkv=0), "shape"), (dict(layers=0), "shape"), (dict(dtype=2), "dtype"), (dict(kind=2), "kind"), (dict(table=0), "null"), (dict(status=0), "null"),
       (dict(kcodes=4097), "aligned"), (dict(vtail=4104), "aligned")]


def _error():
    from kvquant._lib import lib
    return lib.odmkv_last_error().decode()


@pytest.mark.parametrize("change,says", BAD, ids=[next(iter(c)) + "=" + str(next(iter(c.values()))) for c, _ in BAD])
def test_a_bad_cache_is_refused_everywhere(change, says):
    from kvquant._lib import lib
    p, good = C.byref(_pages(**change)), C.byref(_pages())
    for call in (lambda: lib.odmkv_pages_init(p, None), lambda: lib.odmkv_pages_extend(p, None, None, 1, 1, None),
                 lambda: lib.odmkv_pages_write(p, 0, 4096, 0, 0, 128, 4096, 0, 0, 128, 1, None), lambda: lib.odmkv_pages_read(p, 0, 4096, 4096, 0, 1, None),
                 lambda: lib.odmkv_pages_reorder(p, 4096, None, 4096, 1 << 20, None), lambda: lib.odmkv_pages_select(good, p, 4096, 4096, 1 << 20, None),
                 lambda: lib.odmkv_pages_truncate(p, None, None, 0, None, None), lambda: lib.odmkv_pages_compact(p, good, 4096, 1 << 20, None)):
        assert call() == -1 and says in _error(), _error()


def test_bad_arguments_are_refused():
    from kvquant._lib import lib
    p = C.byref(_pages())
    few = (C.c_int32 * 3)(1, 2, 3)
    many = C.byref(_pages(rows=600))
    assert lib.odmkv_pages_extend(p, None, None, -1, 1, None) == -1
    assert lib.odmkv_pages_extend(p, None, None, 2, 1, None) == -1
    assert lib.odmkv_pages_extend(p, 4096, few, 0, 3, None) == -1 and "from the device and from the host" in _error()
    assert lib.odmkv_pages_extend(many, None, (C.c_int32 * 600)(), 0, 3, None) == -1 and "600" in _error()
    assert lib.odmkv_pages_write(p, 2, 4096, 0, 0, 128, 4096, 0, 0, 128, 1, None) == -1 and "layer" in _error()
    assert lib.odmkv_pages_write(p, 0, 0, 0, 0, 128, 4096, 0, 0, 128, 1, None) == -1 and "null" in _error()
    assert lib.odmkv_pages_write(p, 0, 4096, 0, 0, 100, 4096, 0, 0, 128, 1, None) == -1 and "aligned" in _error()
    assert lib.odmkv_pages_write(p, 0, 4096, 0, 0, 128, 4104, 0, 0, 128, 1, None) == -1 and "aligned" in _error()
    assert lib.odmkv_pages_write(p, 0, 4096, 0, 0, 128, 4096, 0, 0, 128, -1, None) == -1
    assert lib.odmkv_pages_write(p, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None) == 0                           # nothing to store
    assert lib.odmkv_pages_read(p, 0, 4096, 4096, 3, 1, None) == -1 and lib.odmkv_pages_read(p, 0, 0, 4096, 0, 1, None) == -1
    assert lib.odmkv_pages_read(p, 0, 0, 0, 0, 0, None) == 0
    assert lib.odmkv_pages_reorder(p, None, None, 4096, 1 << 20, None) == -1 and lib.odmkv_pages_reorder(p, 4096, few, 4096, 1 << 20, None) == -1
    assert lib.odmkv_pages_reorder(p, 4096, None, 4096, 8, None) == -2 and "workspace" in _error()
    assert lib.odmkv_pages_truncate(p, None, None, -1, None, None) == -1
    other = _pages(kcodes=8192)
    assert lib.odmkv_pages_select(p, C.byref(other), 4096, 4096, 1 << 20, None) == -1 and "share" in _error()
    assert lib.odmkv_pages_select(p, p, 4096, 4096, 1 << 20, None) == -1 and "rows of their own" in _error()
    assert lib.odmkv_pages_compact(p, p, 4096, 1 << 20, None) == -1 and "share memory" in _error()
    assert lib.odmkv_pages_compact(p, C.byref(_pages(rows=2)), 4096, 1 << 20, None) == -1
    apart = C.byref(_pages(**{n: 8192 for n in ("kcodes", "vcodes", "kscale", "vscale", "ktail", "vtail", "table", "length", "start", "slot", "refs", "status")}))
    assert lib.odmkv_pages_compact(p, apart, 4096, 8, None) == -2


def test_bad_attention_is_refused():
    from kvquant._lib import Attend, lib
    pages = _pages()

    def call(**change):
        a = Attend(C.pointer(pages), 4096, 1024, 128, 1024, 4096, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 8, 0, 100, 0.1, 0.0)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.odmkv_pages_attend(C.byref(a), None)

    for change, says in ((dict(layer=2), "layer"), (dict(Hq=7), "heads"), (dict(Hq=36), "heads"), (dict(Hq=0), "heads"), (dict(L=-1), "length"), (dict(window=-1), "length"),
                         (dict(max_length=-1), "length"), (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"), (dict(cap=float("nan")), "cap"), (dict(q=0), "null"),
                         (dict(out=0), "null"), (dict(q=4100), "aligned"), (dict(q_stride_l=100), "aligned")):
        assert call(**change) == -1 and says in _error(), (change, _error())
    assert call(L=0) == 0
    assert lib.odmkv_pages_attend(None, None) == -1
    # a call whose blocks are shared out needs room for the shares
    need = lib.odmkv_pages_attend_workspace_bytes(C.byref(pages), 8, 1, 100000)
    assert need > 0 and call(max_length=100000) == -2 and call(max_length=100000, workspace=4096, workspace_bytes=need - 1) == -2
    assert lib.odmkv_pages_attend_workspace_bytes(None, 8, 1, 100) == 0


def test_python_refusals_without_a_gpu():
    from kvquant import PagedKVCache
    for args, kw in (((0, 1, 10), {}), ((1025, 1, 10), {}), ((1, 0, 10), {}), ((1, 1, 0), {}), ((1, 1, 10), dict(layers=0)), ((1, 1, 10), dict(pages=-1)),
                     ((1, 1, 10), dict(kind="int4")), ((1, 1, 10), dict(dtype=torch.float32)), ((1, 1, 10), dict(head_dim=64)), ((1, 1, 10), dict(layers=70000))):
        with pytest.raises(ValueError):
            PagedKVCache(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        PagedKVCache(1, 1, 10, device="cpu")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_the_plain_statement(kind):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(2, 200, 128, generator=g) * 3).half()
    held = plain.held(x, kind)
    assert torch.equal(held[:, 192:], x[:, 192:].double())
    blocks = x[:, :192].double().view(2, 3, 64, 128)
    a = blocks.abs().amax(dim=(-1, -2))
    s = plain.scale_of(a, plain.TOP[kind])
    assert bool((s >= a / plain.TOP[kind]).all()) and bool((s <= a / plain.TOP[kind] * (1 + 2.0 ** -7)).all())
    codes = held[:, :192].view(2, 3, 64, 128) / s[..., None, None]
    if kind == "int8":
        assert torch.equal(codes, codes.round()) and float(codes.abs().max()) <= 127
        # the largest step is a scale; a rounding is off by half of it at most
        assert bool(((held[:, :192].view(2, 3, 64, 128) - blocks).abs() <= s[..., None, None] / 2).all())
    else:
        assert torch.equal(codes, codes.float().to(torch.float8_e4m3fn).double())
        # half a step of e4m3 is 2^-4 of the value, and 2^-10 below its normal numbers
        assert bool(((codes - blocks / s[..., None, None]).abs() <= torch.maximum(codes.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10))).all())


@pytest.mark.parametrize("mask", [object(), torch.ones(1, 9, dtype=torch.bool), torch.ones(1, 1, 2, 8, dtype=torch.bool), torch.ones(1, 1, 2, 9, dtype=torch.bool)],
                         ids=["no tensor", "two dims", "another length", "not causal"])
def test_masks_that_the_pages_cannot_answer_are_refused(mask):
    from kvquant.attention_patch import _paged_attention
    with pytest.raises(RuntimeError, match="cannot be answered from the paged cache"):
        _paged_attention((None, 0, 9), None, torch.zeros(1, 2, 2, 128), mask, 0.0, {})
