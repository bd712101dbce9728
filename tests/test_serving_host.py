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


def _prompt(**change):
    from kvquant._lib import PromptAttend, lib
    a = PromptAttend(*[4096, 1024, 128, 1024] * 3, 4096, 4096, 0, 0, 0, 0, 0, 0, 2, 1000, 1000, 8, 4, 1, 0, 0.1, 0.0)
    for name, value in change.items():
        setattr(a, name, value)
    return lib.odmkv_prompt_attend(C.byref(a), None)


def test_bad_prompts_are_refused():
    from kvquant._lib import lib
    nan, inf = float("nan"), float("inf")
    for change, says in ((dict(dtype=2), "dtype"), (dict(rows=0), "shape"), (dict(L=-1), "shape"), (dict(T=-1), "shape"), (dict(L=(1 << 26) + 1), "shape"), (dict(Hkv=0), "heads"),
                         (dict(Hq=7), "heads"), (dict(Hq=0), "heads"), (dict(window=-1), "window"), (dict(window=5, causal=0), "window"), (dict(cap=-1.0), "cap"), (dict(cap=nan), "cap"),
                         (dict(cap=inf), "cap"), (dict(cap=1e-38), "cap"), (dict(key_offsets=4096), "offsets"), (dict(q=0), "null"), (dict(k=0), "null"), (dict(v=0), "null"),
                         (dict(out=0), "null"), (dict(q=4100), "aligned"), (dict(out=4104), "aligned"), (dict(k_stride_t=100), "aligned"),
                         (dict(rows=1 << 20, L=1 << 26), "too many"), (dict(Hq=65532, L=1 << 26), "too many")):
        assert _prompt(**change) == -1 and says in _error(), (change, _error())
    assert _prompt(L=0) == 0                                                             # nobody asks
    assert lib.odmkv_prompt_attend(None, None) == -1 and "null" in _error()
    # few queries over many keys: their blocks are shared out, and the shares need room
    few = dict(rows=1, L=2, T=50000)
    need = lib.odmkv_prompt_attend_workspace_bytes(0, 1, 8, 4, 2, 50000, 1, 0, 0.0)
    assert need > 0 and _prompt(**few) == -2 and _prompt(**few, workspace=4096, workspace_bytes=need - 1) == -2 and _prompt(**few, workspace=4100, workspace_bytes=need) == -2
    assert lib.odmkv_prompt_attend_workspace_bytes(0, 0, 8, 4, 2, 50000, 1, 0, 0.0) == 0 and lib.odmkv_prompt_attend_workspace_bytes(0, 1, 7, 4, 2, 50000, 1, 0, 0.0) == 0


def test_python_refuses_prompts_without_a_gpu():
    import torch
    from kvquant import prompt_attention
    q = torch.zeros(1, 4, 5, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        prompt_attention(q, q, q)
    with pytest.raises(ValueError, match="queries must be"):
        prompt_attention(None, q, q)


@pytest.mark.parametrize("change,says", BAD, ids=[next(iter(c)) + "=" + str(next(iter(c.values()))) for c, _ in BAD])
def test_a_plan_of_a_bad_cache_is_refused(change, says):
    from kvquant._lib import lib
    assert lib.odmkv_pages_plan(C.byref(_pages(**change)), 4096, 1 << 20, None) == -1 and says in _error(), _error()


def test_bad_plans_are_refused():
    from kvquant._lib import Attend, lib
    pages = _pages()
    p = C.byref(pages)
    need = lib.odmkv_pages_plan_bytes(3)
    assert need >= 4 * (1 + 4 * 3 + 3) and lib.odmkv_pages_plan_bytes(0) == 0
    assert lib.odmkv_pages_plan(p, 0, need, None) == -1 and lib.odmkv_pages_plan(p, 4100, need, None) == -1 and "aligned" in _error()
    assert lib.odmkv_pages_plan(p, 4096, need - 1, None) == -2 and "too small" in _error()
    a = Attend(C.pointer(pages), 4096, 1024, 128, 1024, 4096, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 8, 0, 100, 0.1, 0.0, 4096)
    need = lib.odmkv_pages_attend_shared_workspace_bytes(p, 8, 1, 100)
    assert need > lib.odmkv_pages_attend_workspace_bytes(p, 8, 1, 100)
    assert lib.odmkv_pages_attend(C.byref(a), None) == -2 and "workspace" in _error()
    a.workspace, a.workspace_bytes = 4096, need - 1
    assert lib.odmkv_pages_attend(C.byref(a), None) == -2
    assert lib.odmkv_pages_attend_shared_workspace_bytes(None, 8, 1, 100) == 0
    # what takes the ordinary way takes its workspace
    assert lib.odmkv_pages_attend_shared_workspace_bytes(p, 8, 40, 9000) == lib.odmkv_pages_attend_workspace_bytes(p, 8, 40, 9000)


# ---- headers that the host compiles as the entry points and kernels do
def _compiled(folder, name, source):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (folder / f"{name}.cpp").write_text(f'#include "{name}.h"\n{source}\n')
    subprocess.run(["g++", "-O2", "-fwrapv", "-shared", "-fPIC", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(root, "odm-kv_amd", "csrc"),
                    str(folder / f"{name}.cpp"), "-o", str(folder / f"{name}.so")], check=True)
    return C.CDLL(str(folder / f"{name}.so"))


@pytest.fixture(scope="module")
def span_of(tmp_path_factory):
    """What offsets say, where nobody on the host has seen them (csrc/spans.h)."""
    f = _compiled(tmp_path_factory.mktemp("spans"), "spans",
                  'extern "C" void span(int first, int last, int all, int* to) { const Span s = span_of(first, last, all); to[0] = s.begin; to[1] = s.n; }').span
    f.argtypes, f.restype = [C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int)], None

    def call(first, last, all):
        to = (C.c_int * 2)()
        f(first, last, all, to)
        return to[0], to[1]
    return call


def test_spans_of_any_offsets_stay_within_what_there_is(span_of):
    """Offsets that ascend are taken as they are, within the tensors; what does not ascend is empty; both ends of 32 bits among them."""
    some = [-2 ** 31, -2 ** 31 + 1, -2 ** 30, -1, 0, 1, 63, 64, 99, 100, 101, 2 ** 26, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    for all in (0, 1, 100, 2 ** 26):
        for first in some:
            for last in some:
                begin = min(max(first, 0), all)
                want = begin, max(min(max(last, 0), all) - begin, 0)
                assert span_of(first, last, all) == want, (first, last, all)


def test_partial_results_lie_apart_and_on_16_bytes(tmp_path):
    """Any number of results, odd ones among them: results begin on 16 bytes, nothing lies in another's place, and all of it within what is asked for."""
    f = _compiled(tmp_path, "parts", 'extern "C" void places(size_t parts, size_t common, size_t* to) { const PartPlaces p = part_places(parts, common); to[0] = p.lse; '
                  'to[1] = p.common_out; to[2] = p.common_lse; to[3] = p.floats; }').places
    f.argtypes, f.restype = [C.c_size_t, C.c_size_t, C.POINTER(C.c_size_t)], None
    for parts in (0, 1, 2, 3, 4, 5, 21, 63, 3 * 7 * 5, 2 ** 20 + 1, 2 ** 26 + 3):
        for common in (0, 1, 2, 3, 128 * 5 + 21, 2 ** 25 + 1):
            to = (C.c_size_t * 4)()
            f(parts, common, to)
            lse, out, common_lse, floats = to
            assert lse % 4 == 0 and out % 4 == 0, (parts, common)
            assert lse >= 128 * parts and out >= lse + parts and common_lse >= out + 128 * common and floats >= common_lse + common, (parts, common)
            assert floats <= 129 * (parts + common) + 8


def test_what_a_call_would_have_to_record():
    import torch
    from torch.autograd import forward_ad
    from kvquant.paged_cache import _recorded
    x = torch.ones(3)
    y = x.clone().requires_grad_()
    assert not _recorded(x, None, 5) and _recorded(x, y) and _recorded(2 * y)
    with torch.no_grad():
        assert not _recorded(x, y)
    with forward_ad.dual_level(), torch.no_grad():
        assert not _recorded(x, y) and _recorded(x, forward_ad.make_dual(x, torch.ones(3)))
