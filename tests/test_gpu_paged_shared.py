"""GPU: attention over blocks that rows have in common, read once for all of them, against the definition of each row by itself; the plan that says which blocks those are."""
import pytest
import torch

import test_gpu_paged_cache as paged
from test_gpu_paged_cache import DEV, _cache, _queries, _rows

pytestmark = pytest.mark.gpu


def _samples(seed, prompts, parents, fresh, H, dtype, kind, room=0):
    """A batch of rows that go on from prompts of the given lengths (parents: row -> prompt) by `fresh` tokens each, and what its rows hold."""
    k, v = _rows(seed, len(prompts), H, max(prompts), dtype)
    k1, v1 = _rows(seed + 1, len(parents), H, max(max(fresh), 1), dtype)
    pages = sum(n // 64 for n in prompts) + sum((n + room) // 64 + 2 for n in fresh)
    c = _cache(len(prompts), H, max(prompts) + max(fresh) + room + 1, pages=pages, kind=kind, dtype=dtype)
    c.append(k.to(DEV), v.to(DEV), prompts)
    batch = c.select(parents)
    c.release()
    batch.append(k1.to(DEV), v1.to(DEV), fresh)
    rows = [tuple(torch.cat((x[g, :, :prompts[g]], y[b, :, :fresh[b]]), dim=1) for x, y in ((k, k1), (v, v1))) for b, g in enumerate(parents)]
    return batch, rows


def _check_attend(c, rows, kind, q, **how):
    """The check of the ordinary calls, of the calls that read what is in common once."""
    class Shared:
        def attend(self, *args, **kw):
            return c.attend(*args, shared=True, **kw)
    paged._check_attend(Shared(), rows, kind, q, **how)


def _plan(c):
    """The plan of a cache as a list of (rows, blocks), and every row's blocks."""
    B, plan = c.batch, c._plan.tolist()
    common, group, member, order = (plan[1 + i * B:1 + (i + 1) * B] for i in range(4))
    groups = []
    for g in range(plan[0]):
        begin, members, blocks, slot = plan[1 + 4 * B + 4 * g:5 + 4 * B + 4 * g]
        rows = order[begin:begin + members]
        assert slot == int(c.slot[rows[0]])
        for i, b in enumerate(rows):
            assert group[b] == g and member[b] == i and common[b] == blocks
        groups.append((rows, blocks))
    assert sum(len(rows) for rows, _ in groups) == sum(n > 0 for n in common)
    return groups


def _plan_of_tables(c):
    """The same from the tables."""
    table, slot, length = c.table.tolist(), c.slot.tolist(), c.length.tolist()
    held = [table[slot[b]][:length[b] // 64] for b in range(c.batch)]
    groups = {}
    for b, pages in enumerate(held):
        if pages:
            groups.setdefault(pages[0], []).append(b)
    out = []
    for rows in groups.values():
        if len(rows) > 1:
            first = held[rows[0]]
            out.append((rows, min(next((j for j, (x, y) in enumerate(zip(first, held[b])) if x != y), min(len(first), len(held[b]))) for b in rows)))
    return out


CASES = [([200], [0, 0], [0, 0], 4, 1, 1), ([64], [0] * 8, [5, 0, 1, 64, 63, 130, 7, 70], 8, 2, 1), ([63], [0, 0, 0], [1, 70, 3], 4, 2, 1), ([700], [0] * 4, [1] * 4, 28, 4, 2),
         ([1000], [0] * 17, list(range(17)), 8, 1, 2), ([640, 300, 129], [0, 1, 0, 2, 1, 0, 2, 0], [3, 200, 0, 64, 1, 80, 6, 33], 6, 2, 1),
         ([300, 300], [0, 1], [4, 5], 4, 2, 1), ([300, 400], [1, 1, 0], [4, 5, 6], 4, 4, 5), ([150], [0] * 100, [b % 70 for b in range(100)], 4, 1, 1),
         ([5000], [0] * 33, [b * 3 for b in range(33)], 8, 2, 1), ([130, 64], [0] * 40 + [1] * 30, [b % 3 for b in range(70)], 8, 1, 2)]


@pytest.mark.parametrize("kind,dtype", [("int8", torch.float16), ("e4m3", torch.bfloat16), ("int8", torch.bfloat16)])
@pytest.mark.parametrize("prompts,parents,fresh,Hq,H,L", CASES, ids=[f"{c[0]}x{len(c[1])}-{c[3]}-{c[4]}-{c[5]}" for c in CASES])
def test_rows_in_common(prompts, parents, fresh, Hq, H, L, kind, dtype):
    c, rows = _samples(len(parents), prompts, parents, fresh, H, dtype, kind)
    _check_attend(c, rows, kind, _queries(7, len(parents), Hq, L, dtype))
    assert _plan(c) == _plan_of_tables(c)


ODD = [([200], [0] * 3, [1, 0, 5], 7, 1, 1), ([130], [0] * 5, [3, 64, 0, 1, 70], 5, 1, 1), ([300, 130], [0, 1, 0, 1, 1, 0, 0], [2, 3, 64, 9, 1, 0, 5], 3, 1, 3),
       ([150], [0] * 151, [b % 70 for b in range(151)], 7, 1, 1), ([130], [0] * 201, [b % 3 for b in range(201)], 3, 1, 2), ([500], [0] * 79, [b % 66 for b in range(79)], 5, 1, 3),
       ([70, 200], [b % 2 for b in range(111)], [b % 5 for b in range(111)], 10, 2, 1), ([64], [0] * 1023, [1] * 1023, 1, 1, 1), ([64], [0] * 1024, [1] * 1024, 3, 1, 1)]


@pytest.mark.parametrize("prompts,parents,fresh,Hq,H,L", ODD, ids=[f"{c[0]}x{len(c[1])}-{c[3]}-{c[4]}-{c[5]}" for c in ODD])
def test_odd_counts_of_queries(prompts, parents, fresh, Hq, H, L):
    """One kv-head and odd numbers of rows and query heads: partial results whose number is no multiple of four, and more than 1024 queries, of which a workgroup puts four together."""
    for dtype in (torch.float16, torch.bfloat16):
        c, rows = _samples(len(parents), prompts, parents, fresh, H, dtype, "int8")
        _check_attend(c, rows, "int8", _queries(7, len(parents), Hq, L, dtype))
        assert _plan(c) == _plan_of_tables(c)


MASKS = {"cap": dict(softcap=20.0), "large cap": dict(softcap=3000.0), "window inside": dict(window=30), "window across": dict(window=200), "bias": dict(slopes=0.25),
         "scaling": dict(scaling=-0.05), "prefix": dict(prefix=[130, 0, 500, 400, 1]), "starts": dict(starts=[70, 0, 256, 310, 10 ** 6]), "starts of each": dict(starts="each"),
         "counts": dict(counts=[2, 0, 1, 2, 0]), "all": dict(softcap=30.0, slopes=0.1, window=290, prefix=[100, 400, 3, 0, 290], starts=[5, 200, 0, 64, 0], counts=[1, 2, 2, 0, 2])}


@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("Hq,H", [(6, 2), (8, 1)])
def test_masks(mask, Hq, H):
    how, dtype = dict(MASKS[mask]), torch.bfloat16 if Hq == 6 else torch.float16
    c, rows = _samples(3, [280], [0] * 5, [3, 60, 130, 2, 40], H, dtype, "int8")
    for name in ("prefix", "starts", "counts"):
        if name in how and how[name] != "each":
            how[name] = torch.tensor(how[name], dtype=torch.int32)
    if "starts" in how and not isinstance(how["starts"], torch.Tensor):
        how["starts"] = torch.randint(0, 320, (5, 2), generator=torch.Generator().manual_seed(2)).int()
    if "slopes" in how:
        how["slopes"] = how["slopes"] * torch.linspace(0.1, 1, Hq)
    _check_attend(c, rows, "int8", _queries(5, 5, Hq, 2, dtype), **how)


def test_a_prompt_of_many_blocks():
    """More blocks a share than are looked up at a time, several tiles of queries; nothing of their own for some rows."""
    c, rows = _samples(4, [20000], [0] * 9, [0, 1, 64, 0, 300, 2, 0, 65, 9], 1, torch.float16, "int8")
    _check_attend(c, rows, "int8", _queries(5, 9, 8, 2, torch.float16))


def test_more_queries_than_sixteen_take_the_ordinary_way():
    c, _ = _samples(6, [300], [0] * 3, [5, 6, 7], 2, torch.float16, "int8")
    q = _queries(5, 3, 8, 5, torch.float16).to(DEV)
    for x, y in zip(c.attend(0, q, shared=True, return_lse=True), c.attend(0, q, return_lse=True)):
        assert torch.equal(x, y)
    one = c.select([1])
    for x, y in zip(one.attend(0, q[:1, :, :1], shared=True, return_lse=True), one.attend(0, q[:1, :, :1], return_lse=True)):
        assert torch.equal(x, y)
    odd = torch.zeros(3, 8, 1, 130, dtype=torch.float16, device=DEV)[..., 1:129]        # (a copy is made: not by the native call)
    odd.copy_(q[:, :, :1])
    assert torch.equal(c.attend(0, odd, shared=True), c.attend(0, q[:, :, :1], shared=True))


def test_no_plan_is_kept_that_nobody_reads():
    """More queries than sixteen, and a batch of one row, take the ordinary way: no plan is made, and they can be captured without one."""
    c, rows = _samples(6, [300], [0] * 3, [5, 6, 7], 2, torch.float16, "int8")
    wide, one = _queries(5, 3, 8, 5, torch.float16), c.select([1])
    for cache, q, held in ((c, wide, rows), (one, wide[:1, :, :1], rows[1:2])):
        _check_attend(cache, held, "int8", q)
        assert cache._plan is None
        q = q.to(DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = cache.attend(0, q, shared=True)
        for _ in range(3):
            graph.replay()
            want = cache.attend(0, q, longest=cache.max_tokens)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        cache.reorder(list(range(cache.batch)))
        assert cache._plan is None
    _check_attend(c, rows, "int8", _queries(5, 3, 8, 4, torch.float16))                    # sixteen
    assert _plan(c) == _plan_of_tables(c) == [([0, 1, 2], 4)]
    _check_attend(c, rows, "int8", wide)


def test_the_plan_follows_the_rows():
    """Beams that are reordered, cut into what they share, freed, forked and compacted: the plan is what the tables say, the attention what the rows hold."""
    B, H, dtype = 6, 2, torch.bfloat16
    c, rows = _samples(8, [200], [0] * B, [0] * B, H, dtype, "int8", room=400)
    q = _queries(9, B, 8, 1, dtype)
    c.attend(0, q.to(DEV), shared=True)
    g = torch.Generator().manual_seed(10)
    k, v = _rows(11, B, H, 300, dtype)
    for step in range(8):
        parents = torch.randint(0, B, (B,), generator=g)
        c.reorder(parents.to(DEV) if step % 2 else parents.tolist())
        rows = [rows[b] for b in parents.tolist()]
        assert _plan(c) == _plan_of_tables(c)
        n = 40
        at = step * n % 260
        c.append(k[:, :, at:at + n].to(DEV), v[:, :, at:at + n].to(DEV))
        rows = [tuple(torch.cat((x, y[b, :, at:at + n]), dim=1) for x, y in zip(row, (k, v))) for b, row in enumerate(rows)]
        _check_attend(c, rows, "int8", q)
        assert _plan(c) == _plan_of_tables(c)
    c.truncate(130, rows=[2])                                                # into what it shares
    c.free([4])
    import paged_rows as plain
    rows[2], rows[4] = (tuple(plain.cut(x, n, "int8") for x in rows[b]) for b, n in ((2, 130), (4, 0)))
    assert _plan(c) == _plan_of_tables(c)
    _check_attend(c, rows, "int8", q)
    forked = c.select([0, 0, 3, 3, 3, 2])
    _check_attend(forked, [rows[b] for b in (0, 0, 3, 3, 3, 2)], "int8", q)
    assert _plan(forked) == _plan_of_tables(forked) and _plan(c) == _plan_of_tables(c)
    forked.release()
    packed = c.compacted()
    _check_attend(packed, rows, "int8", q)
    assert _plan(packed) == _plan_of_tables(packed)


def test_many_rows_and_no_rows_in_common():
    c, rows = _samples(12, [70], [0] * 300, [1] * 300, 1, torch.float16, "int8")
    _check_attend(c, rows, "int8", _queries(5, 300, 2, 1, torch.float16))
    assert _plan(c) == [(list(range(300)), 1)]
    k, v = _rows(13, 5, 2, 500, torch.float16)
    lengths = [500, 0, 64, 63, 400]
    c = _cache(5, 2, 600)
    c.append(k.to(DEV), v.to(DEV), lengths)
    _check_attend(c, [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(lengths)], "int8", _queries(5, 5, 8, 1, torch.float16))
    assert _plan(c) == []


def test_captured_beams():
    """A step of beams in one graph: every replay's plan is of the rows as they are then, with eager work in between."""
    B, H, dtype, n = 4, 2, torch.bfloat16, 62
    eager, captured = (_samples(14, [260], [0] * B, [0] * B, H, dtype, "int8", room=400)[0] for _ in range(2))
    q = _queries(15, B, 8, 1, dtype).to(DEV)
    k, v = (x.to(DEV) for x in _rows(16, B, H, 8, dtype))
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            captured.attend(0, q, shared=True)
    captured.attend(0, q, shared=True)
    eager.attend(0, q, shared=True)
    parents = torch.arange(B, device=DEV)
    ks, vs = k[:, :, :1].clone(), v[:, :, :1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.reorder(parents)
        captured.extend(1)
        captured.write(0, ks, vs)
        out, lse = captured.attend(0, q, shared=True, return_lse=True)
    g = torch.Generator().manual_seed(17)
    for i in range(6):
        order = torch.randint(0, B, (B,), generator=g)
        parents.copy_(order)
        ks.copy_(k[:, :, i:i + 1])
        vs.copy_(v[:, :, i:i + 1])
        graph.replay()
        eager.reorder(order.tolist())
        eager.append(k[:, :, i:i + 1], v[:, :, i:i + 1])
        want, want_lse = eager.attend(0, q, shared=True, return_lse=True, longest=captured.max_tokens)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and _plan(captured) == _plan(eager), i
        if i == 3:                                                           # rows are moved between the replays as well
            for c in (eager, captured):
                c.truncate([200, 128, 250, 251])
    captured.refresh()


def test_rows_that_a_captured_call_moves_before_there_is_a_plan():
    B, H, dtype = 4, 2, torch.float16
    c, rows = _samples(18, [300], [0] * B, [70, 5, 9, 80], H, dtype, "int8", room=10)
    graph = torch.cuda.CUDAGraph()
    parents = torch.tensor([1, 1, 3, 3], device=DEV)
    with torch.cuda.graph(graph):
        c.reorder(parents)
    c._bounds[:] = [c.max_length] * B
    q = _queries(19, B, 4, 1, dtype)
    _check_attend(c, rows, "int8", q)
    graph.replay()
    rows = [rows[b] for b in (1, 1, 3, 3)]
    _check_attend(c, rows, "int8", q)
    assert _plan(c) == _plan_of_tables(c)
    parents.copy_(torch.tensor([3, 2, 1, 0]))
    graph.replay()
    _check_attend(c, rows[::-1], "int8", q)
    assert _plan(c) == _plan_of_tables(c)


def test_two_calls_give_the_same_bits():
    c, _ = _samples(20, [2000], [0] * 12, list(range(12)), 2, torch.bfloat16, "e4m3")
    q = _queries(21, 12, 8, 2, torch.bfloat16).to(DEV)
    first = c.attend(0, q, shared=True, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = c.attend(0, q, shared=True, return_lse=True)
    side.synchronize()
    for x, y in zip(first, second):
        assert torch.equal(x, y)


@pytest.mark.parametrize("n", [1, 64, 3000])
def test_a_row_by_itself(n):
    """A batch of one row, and rows of which only one holds anything: there is nothing in common, whatever is asked for."""
    k, v = (x.to(DEV) for x in _rows(40, 1, 2, n, torch.bfloat16))
    one = _cache(1, 2, n + 4, dtype=torch.bfloat16)
    one.append(k, v)
    q = _queries(41, 1, 8, 1, torch.bfloat16)
    for a, b in zip(one.attend(0, q.to(DEV), return_lse=True), one.attend(0, q.to(DEV), shared=True, return_lse=True)):
        assert torch.equal(a, b)
    one.truncate(n)
    one.reorder([0])
    _check_attend(one, [(k[0].cpu(), v[0].cpu())], "int8", q)
    three = one.select([0, 0, 0])
    three.free([0, 2])
    q = _queries(42, 3, 8, 1, torch.bfloat16).to(DEV)
    want, got = (three.attend(0, q, **how) for how in (dict(), dict(shared=True)))
    # (each is rounded to bf16 once, by 2^-8 of itself at most; what else differs is the order of sums in 32 bits and weights in fp16, less than a step of either)
    assert not got[0].any() and not got[2].any() and (want[1].float() - got[1].float()).abs().max() <= 2 * 2.0 ** -8 * want[1].float().abs().max()


@pytest.mark.parametrize("n", [1, 64, 3000])
def test_rows_of_which_one_holds_anything(n):
    """A plan that there was when the others were freed, and one made behind that: every element and log-sum-exp is the definition's, empty rows give 0 and -inf."""
    k, v = (x.to(DEV) for x in _rows(40, 1, 2, n, torch.bfloat16))
    one = _cache(1, 2, n + 4, dtype=torch.bfloat16)
    one.append(k, v)
    q = _queries(42, 3, 8, 1, torch.bfloat16)
    mine, empty = ((x[0].cpu() for x in (k, v)), (x[0, :, :0].cpu() for x in (k, v)))
    mine, empty = tuple(mine), tuple(empty)
    for before in (True, False):
        three = one.select([0, 0, 0])
        if before:
            _check_attend(three, [mine] * 3, "int8", q)
        three.free([0, 2])
        _check_attend(three, [empty, mine, empty], "int8", q)
        out, lse = three.attend(0, q.to(DEV), shared=True, return_lse=True)
        assert not out[[0, 2]].any() and bool((lse[[0, 2]] == -torch.inf).all()) and _plan(three) == []
        three.release()
