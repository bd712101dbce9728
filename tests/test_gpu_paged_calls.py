"""GPU: calls of the paged 8-bit cache that its documentation allows and that are easily missed: odd strides, limits in replays, batches that are dropped, graphs of long rows."""
import gc

import pytest
import torch

import paged_rows as plain
from test_gpu_paged_cache import DEV, _cache, _check_attend, _filled, _holds, _pages_add_up, _queries, _rows

pytestmark = pytest.mark.gpu


def test_strides_of_single_rows_mean_nothing():
    """Dimensions of one with strides that are no multiple of 8: one token, one head, one row."""
    k, v = _rows(1, 1, 1, 70, torch.float16)
    c = _filled(k, v, [70], "int8")
    q = _queries(1, 1, 4, 1, torch.float16)
    odd = torch.zeros(4 * 128, dtype=torch.float16, device=DEV).as_strided((1, 4, 1, 128), (3, 128, 5, 1)).copy_(q)
    assert torch.equal(c.attend(0, odd), c.attend(0, q.to(DEV)))
    c.extend(1)
    one = torch.zeros(128, dtype=torch.float16, device=DEV).as_strided((1, 1, 1, 128), (9, 7, 5, 1))
    one.copy_(k[:, :, :1])
    c.write(0, one, one)
    _holds(c, 0, [tuple(torch.cat([x[0], k[0, :, :1]], dim=1) for x in (k, v))], "int8")


def test_a_layer_that_has_not_stored_its_tokens_is_not_read():
    k, v = _rows(1, 2, 1, 70, torch.float16)
    k, v = k.to(DEV), v.to(DEV)
    q = _queries(1, 2, 4, 1, torch.float16).to(DEV)
    c = _cache(2, 1, 300, layers=2)
    c.attend(1, q)                                            # (empty rows see nothing)
    c.extend(70)
    c.write(0, k, v)
    c.attend(0, q)
    for call in (lambda: c.attend(1, q), lambda: c.attend(1, q, return_lse=True, window=5), lambda: c.read(1), lambda: c.attend(1, q[..., ::2])):
        with pytest.raises(ValueError, match="layer 1 has not stored"):
            call()
    for layer in (2, -1):
        with pytest.raises(ValueError, match="of 2"):
            c.attend(layer, q)
    c.write(1, k, v)
    assert torch.equal(c.attend(1, q), c.attend(0, q))
    c.extend(0)                                               # (nothing to store)
    assert torch.equal(c.attend(1, q), c.attend(0, q))
    c.extend([0, 1])
    small = c.compacted()
    for cache in (c, small):
        with pytest.raises(ValueError, match="has not stored"):
            cache.attend(0, q)
        cache.write(0, k[:, :, :1], v[:, :, :1])
        cache.attend(0, q)


@pytest.mark.parametrize("max_tokens", [200, 256, 192])
def test_a_replay_past_max_tokens_is_refused(max_tokens):
    """Rows may have max_tokens, whatever their table has places for; the replay that would pass it changes nothing and is reported."""
    c = _cache(2, 1, max_tokens, pages=20)
    c.extend([max_tokens - 10, 3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(5)
    for n in (max_tokens - 5, max_tokens):
        graph.replay()
        assert c.refresh() == [n, n - max_tokens + 13]
    for _ in range(2):
        graph.replay()
        with pytest.raises(RuntimeError, match="beyond max_tokens"):
            c.refresh()
        assert c.refresh() == [max_tokens, 13]
    c.truncate(max_tokens - 4, rows=[0])
    graph.replay()
    with pytest.raises(RuntimeError, match="beyond max_tokens"):
        c.refresh()
    c.truncate(max_tokens - 5, rows=[0])
    graph.replay()
    assert c.refresh() == [max_tokens, 18]
    _pages_add_up(c)


@pytest.mark.parametrize("first", ["selected", "original"])
def test_a_dropped_batch_gives_its_pages_back(first):
    """Without `release`: its pages are free again for the other batches over the pool, which can be compacted."""
    k, v = _rows(1, 2, 2, 200, torch.float16)
    c = _cache(2, 2, 400, pages=8)
    c.append(k.to(DEV), v.to(DEV), [200, 130])
    other = c.select([0, 0, 1])
    other.extend(64)                                          # three pages, all that are left
    other.write(0, k[:1, :, :64].expand(3, 2, 64, 128).to(DEV), v[:1, :, :64].expand(3, 2, 64, 128).to(DEV))
    with pytest.raises(ValueError, match="out of pages"):
        c.extend(64)
    if first == "selected":
        kept, rows = c, [(k[0], v[0]), (k[1, :, :130], v[1, :, :130])]
        del other
    else:
        kept, rows = other, [tuple(torch.cat([x[b, :, :n], x[0, :, :64]], dim=1) for x in (k, v)) for b, n in ((0, 200), (0, 200), (1, 130))]
        del c, other
    gc.collect()
    assert kept.refresh() == [r[0].shape[1] for r in rows]
    _pages_add_up(kept)
    _holds(kept, 0, rows, "int8")
    if first == "selected":                                   # (the other one holds all eight pages still)
        kept.extend([64, 128])
    small = kept.compacted()
    assert small.pages == int((kept.refs > 0).sum())
    _pages_add_up(small)


def test_a_batch_dropped_while_a_graph_is_captured_is_left_for_later():
    k, v = _rows(2, 1, 1, 130, torch.float16)
    c = _filled(k, v, [130], "int8", pages=4)
    other = c.select([0])
    other.extend(64)
    side = torch.cuda.CUDAGraph()
    with torch.cuda.graph(side):
        del other
        gc.collect()
        c.extend(1)
    for n in (131, 132):
        side.replay()
        torch.cuda.synchronize()
        assert c.length.tolist() == [n]
    assert int((c.refs > 0).sum()) == 3
    assert c.refresh() == [132] and int((c.refs > 0).sum()) == 2
    _pages_add_up(c)


@pytest.mark.parametrize("L", [1, 20])
def test_a_captured_step_is_cut_for_rows_as_long_as_they_may_become(L, monkeypatch):
    """A graph captured over short rows and replayed over long ones shares their blocks out as an eager call does."""
    from kvquant import paged_cache
    cuts, native = [], paged_cache._native

    class Watched:
        paged_write = staticmethod(native.paged_write)

        @staticmethod
        def paged_attend(*args):
            cuts.append(args[9])
            return native.paged_attend(*args)

    monkeypatch.setattr(paged_cache, "_native", Watched)
    m, n = 70, 9000
    k, v = _rows(3, 1, 2, n, torch.float16)
    c = _cache(1, 2, 10000)
    c.append(k[:, :, :m].to(DEV), v[:, :, :m].to(DEV))
    q = _queries(1, 1, 8, L, torch.float16).to(DEV)
    c.attend(0, q)
    c.attend(0, q, longest=5000)
    c.attend(0, q, longest=10 ** 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.attend(0, q, return_lse=True)
        c.attend(0, q, longest=300)
    assert cuts == [m, 5000, 10000, 10000, 300]
    c.append(k[:, :, m:].to(DEV), v[:, :, m:].to(DEV))
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = c.attend(0, q, return_lse=True, longest=10000)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    _check_attend(c, [(k[0], v[0])], "int8", q.cpu())
    for bad in (lambda: c.attend(0, q, longest=-1), lambda: c.attend(0, q[..., ::2], longest=-1)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("L", [3, 40])
def test_queries_in_front_of_a_row_see_no_prefix(L):
    """More queries than tokens: those at i < 0 see nothing, whatever the prefix is."""
    lengths = [2, L + 70, 0]
    k, v = _rows(L, 3, 2, L + 70, torch.float16)
    c = _filled(k, v, lengths, "int8")
    rows = [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(lengths)]
    q = _queries(L, 3, 8, L, torch.float16)
    _check_attend(c, rows, "int8", q, prefix=torch.tensor([2, 50, 7], dtype=torch.int32))
    out, lse = c.attend(0, q.to(DEV), prefix=torch.tensor([2, 50, 7], dtype=torch.int32, device=DEV), return_lse=True)
    assert not out[0, :L - 2].any() and bool((lse[0, :, :L - 2] == float("-inf")).all()) and bool(torch.isfinite(lse[0, :, L - 2:]).all())


def test_select_is_not_captured():
    """Every replay would take its pages again, and lose those of the one before."""
    k, v = _rows(2, 1, 1, 130, torch.float16)
    c = _filled(k, v, [130], "int8")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=DEV)
        for parents in ([0, 0], torch.tensor([0]), torch.zeros(2, dtype=torch.int64)):
            with pytest.raises(RuntimeError, match="captured"):
                c.select(parents)
    graph.replay()
    torch.cuda.synchronize()
    _pages_add_up(c)
    _pages_add_up(c, c.select([0, 0]))


@pytest.mark.parametrize("L", [1, 20])
def test_the_smallest_caps(L):
    """2^-100: every token weighs the same; what is less, 0 in 32 bits among it, is refused and is not taken for no cap."""
    k, v = _rows(2, 1, 1, 130, torch.float16)
    c = _filled(k, v, [130], "int8")
    q = _queries(1, 1, 4, L, torch.float16)
    _check_attend(c, [(k[0], v[0])], "int8", q, softcap=2.0 ** -100)
    for cap in (1e-50, 2.0 ** -101, float("nan")):
        with pytest.raises(ValueError, match="softcap"):
            c.attend(0, q.to(DEV), softcap=cap)


def test_tokens_that_a_replay_stores_can_be_read():
    """Room made by hand, tokens stored by a graph: the host does not know that they are there, and does not say that they are not."""
    m = 60
    k, v = _rows(5, 1, 2, m + 12, torch.float16)
    c = _filled(k[:, :, :m], v[:, :, :m], [m], "int8")
    kn, vn = (torch.zeros(1, 2, 3, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    c.extend(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(0, kn, vn)
    q = _queries(1, 1, 8, 3, torch.float16)
    for n in range(m, m + 12, 3):
        kn.copy_(k[:, :, n:n + 3])
        vn.copy_(v[:, :, n:n + 3])
        c.extend(3)
        graph.replay()
        torch.cuda.synchronize()
        _holds(c, 0, [(k[0, :, :n + 3], v[0, :, :n + 3])], "int8")
        _check_attend(c, [(k[0, :, :n + 3], v[0, :, :n + 3])], "int8", q)
