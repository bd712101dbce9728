"""GPU: the paged 8-bit cache against its definition in 64 bits (tests/paged_rows.py): what it holds, its attention, and its rows and pages."""
import pytest
import torch

import paged_rows as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def _rows(seed, B, H, n, dtype, wide=True):
    """Keys and values with a few wide channels and a spread from token to token."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(B, H, n, 128, generator=g) for _ in range(2))
    if wide:
        k[..., :4] *= 5
        v *= 0.2 + torch.rand(B, H, n, 1, generator=g)
    return k.to(dtype), v.to(dtype)


def _cache(*args, **kw):
    from kvquant import PagedKVCache
    return PagedKVCache(*args, **kw)


def _filled(k, v, lengths, kind, room=200, **kw):
    """A one-layer cache whose row b holds the first lengths[b] tokens of k[b], v[b]."""
    c = _cache(k.shape[0], k.shape[1], max(lengths) + room, kind=kind, dtype=k.dtype, **kw)
    c.append(k.to(DEV), v.to(DEV), lengths)
    return c


def _holds(c, layer, rows, kind):
    """The cache's dense rows are exactly what the definition says of `rows`: a list of (k, v) [H, n, 128]."""
    n = max([k.shape[1] for k, _ in rows] + [1])
    got_k, got_v = c.read(layer, n, dtype=torch.float32)
    assert c.length.tolist() == [k.shape[1] for k, _ in rows]
    for b, (k, v) in enumerate(rows):
        for got, x in ((got_k, k), (got_v, v)):
            want = plain.held(x, kind)
            assert torch.equal(got[b, :, :x.shape[1]].cpu().double(), want), (b, layer)
            assert not got[b, :, x.shape[1]:].any()


def _pages_add_up(*caches):
    """Every page's count of holders is what the tables say, and the counts of free pages follow."""
    want = torch.zeros(caches[0].pages, dtype=torch.int32)
    for c in caches:
        table, slot = c.table.cpu(), c.slot.cpu()
        assert sorted(slot.tolist()) == list(range(c.batch))
        for b, n in enumerate(c.length.tolist()):
            for page in table[slot[b], :n // 64].tolist():
                want[page] += 1
    assert torch.equal(caches[0].refs.cpu(), want)
    free, hint, refused, _ = caches[0].status.tolist()
    assert free == int((want == 0).sum()) and not refused and bool((want[:hint] > 0).all())


# ------------------------------------------------------------------------------------------------ what is held
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 700])
def test_what_is_held(n, dtype, kind):
    k, v = _rows(n, 2, 3, n, dtype)
    c = _filled(k, v, [n, n], kind)
    _holds(c, 0, [(k[b], v[b]) for b in range(2)], kind)
    _pages_add_up(c)
    # in the cache's own type: rounded once
    got = c.read(0)
    for x, y in zip(got, (k, v)):
        for b in range(2):
            assert torch.equal(x[b, :, :n].cpu(), plain.to_type(plain.held(y[b], kind), dtype))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_edges(dtype, kind):
    """Blocks of zeros, one value, values that tie between codes, the largest, the smallest, infinities and NaN; the last block stays a tail."""
    n = 64 * 8 + 5
    k, v = _rows(1, 1, 2, n, dtype)
    for x, h in ((k, 0), (v, 1)):
        x[0, h, :64] = 0
        x[0, h, 64:128] = 0
        x[0, h, 70, 3] = -1.5
        x[0, h, 128:192] = (torch.arange(64 * 128).view(64, 128) % 255 - 127).to(dtype) / 2         # a / 127 is a power of two for int8: ties
        x[0, h, 128, 0] = -63.5
        x[0, h, 192:256] = torch.finfo(dtype).max
        x[0, h, 256:320] = torch.finfo(dtype).smallest_normal * 2.0 ** -5
        x[0, h, 330, 7], x[0, h, 331, 8], x[0, h, 332, 9] = float("inf"), float("-inf"), float("nan")
        x[0, h, 384:448] *= 2.0 ** -20
        x[0, h, 448:512] = x[0, h, 448:449, :1]                                                     # one value throughout
        x[0, h, -2, 5], x[0, h, -1, 6] = float("nan"), float("inf")
    c = _filled(k, v, [n], kind)
    _holds(c, 0, [(k[0], v[0])], kind)
    for x in c.read(0):
        assert torch.isfinite(x).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_how_tokens_arrive_changes_nothing(kind):
    """One at a time, in uneven pieces, all at once, rows of their own lengths and strides: the same bytes."""
    n, dtype = 200, torch.bfloat16
    k, v = _rows(3, 3, 2, n, dtype)
    lengths = [200, 77, 128]
    whole = _filled(k, v, lengths, kind)
    single = _cache(3, 2, 400, kind=kind, dtype=dtype)
    for t in range(n):
        single.append(k[:, :, t:t + 1].to(DEV), v[:, :, t:t + 1].to(DEV), [int(t < m) for m in lengths])
    pieces = _cache(3, 2, 400, kind=kind, dtype=dtype)
    wide = torch.zeros(2, n, 3, 2, 256, dtype=dtype, device=DEV)             # [k or v, T, B, H, 2 D]
    wide[0, ..., 128:], wide[1, ..., 128:] = k.permute(2, 0, 1, 3).to(DEV), v.permute(2, 0, 1, 3).to(DEV)
    at = 0
    for step in (1, 62, 2, 70, 65):
        counts = torch.tensor([max(0, min(step, m - at)) for m in lengths], dtype=torch.int32, device=DEV)
        pieces.extend(counts, bound=step)
        pieces.write(0, wide[0, at:at + step, ..., 128:].permute(1, 2, 0, 3), wide[1, at:at + step, ..., 128:].permute(1, 2, 0, 3))
        at += step
    for c in (whole, single, pieces):
        _holds(c, 0, [(k[b, :, :m], v[b, :, :m]) for b, m in enumerate(lengths)], kind)
        _pages_add_up(c)


def test_rows_that_do_not_start_on_16_bytes():
    k, v = _rows(4, 1, 2, 70, torch.float16)
    c = _cache(1, 2, 200)
    flat = torch.zeros(2 * 70 * 128 + 1, dtype=torch.float16, device=DEV)
    odd = flat[1:].view(1, 2, 70, 128)
    odd.copy_(k)
    c.append(odd, v.to(DEV).transpose(2, 3).contiguous().transpose(2, 3))
    _holds(c, 0, [(k[0], v[0])], "int8")


# ------------------------------------------------------------------------------------------------ attention
def _check_attend(c, rows, kind, q, counts=None, prefix=None, starts=None, slopes=None, **how):
    """cache.attend of q [B, Hq, L, 128] against the definition; rows: (k, v) of every row."""
    B, Hq, L, _ = q.shape
    dtype = q.dtype
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out, lse = c.attend(0, q.to(DEV), counts=dev(counts), prefix=dev(prefix), starts=dev(starts), slopes=dev(slopes), return_lse=True, **how)
    assert out.shape == (B, L, Hq, 128) and out.dtype == dtype
    out, lse = out.cpu().double(), lse.cpu().double()
    args = dict(how)
    args["cap"] = args.pop("softcap", None)
    for b, (k, v) in enumerate(rows):
        n = L if counts is None else int(counts[b])
        st = None if starts is None else (starts[b, :n] if starts.dim() == 2 else starts[b])
        want, wl, tol, tl = plain.attend(q[b, :, :n], plain.held(k, kind), plain.held(v, kind), slopes=slopes,
                                         prefix=None if prefix is None else int(prefix[b]), starts=st, **args)
        got, gl = out[b, :n], lse[b, :, :n]
        assert torch.equal(torch.isinf(gl), torch.isinf(wl)) and torch.isfinite(got).all()
        ok = torch.isfinite(wl)
        assert ((gl - wl).abs()[ok] <= tl[ok] + 2.0 ** -23 * wl.abs()[ok]).all(), float(((gl - wl).abs()[ok] - tl[ok]).max())
        bound = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        off = (got - want).abs()
        assert (off <= bound).all(), (b, float((off / bound.clamp(min=1e-30)).max()))
        assert not out[b, n:].any()


def _queries(seed, B, Hq, L, dtype, size=2.0):
    return (size * torch.randn(B, Hq, L, 128, generator=torch.Generator().manual_seed(seed))).to(dtype)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,L", [(1, 1), (2, 1), (63, 1), (64, 1), (65, 1), (129, 1), (1000, 1), (5000, 1), (66, 3), (700, 4), (17, 17), (64, 64), (200, 33), (333, 333),
                                 (1500, 70)])
@pytest.mark.parametrize("Hq,H", [(8, 2)])
def test_attend(m, L, Hq, H, dtype, kind):
    k, v = _rows(m + L, 1, H, m, dtype)
    _check_attend(_filled(k, v, [m], kind), [(k[0], v[0])], kind, _queries(m, 1, Hq, L, dtype))


@pytest.mark.parametrize("L", [1, 5, 40])
@pytest.mark.parametrize("Hq,H", [(1, 1), (3, 3), (6, 2), (5, 1), (7, 1), (8, 1), (28, 4)])
def test_attend_groups(Hq, H, L):
    k, v = _rows(Hq, 1, H, 300, torch.bfloat16)
    _check_attend(_filled(k, v, [300], "int8"), [(k[0], v[0])], "int8", _queries(L, 1, Hq, L, torch.bfloat16))


MASKS = {
    "cap": dict(softcap=20.0), "small cap": dict(softcap=0.5), "large cap": dict(softcap=3000.0), "window": dict(window=50), "window of one": dict(window=1),
    "window past all": dict(window=100000), "bias": dict(slopes=0.25), "negative bias": dict(slopes=-0.01), "scaling": dict(scaling=0.5),
    "prefix": dict(prefix=[130, 0, 500]), "starts": dict(starts=[70, 0, 64]), "starts of each": dict(starts="each"), "nothing seen": dict(starts=[10 ** 6, 3, 10 ** 9]),
    "all": dict(softcap=30.0, slopes=0.1, window=90, prefix=[100, 400, 3], starts=[5, 200, 0]),
}


@pytest.mark.parametrize("L", [1, 4, 37, 130])
@pytest.mark.parametrize("mask", sorted(MASKS))
def test_attend_masks(mask, L):
    how = dict(MASKS[mask])
    lengths, dtype = [131, 450, 256], torch.float16 if L % 2 else torch.bfloat16
    k, v = _rows(L, 3, 2, 450, dtype)
    if "prefix" in how:
        how["prefix"] = torch.tensor(how["prefix"], dtype=torch.int32)
    if how.get("starts") == "each":
        g = torch.Generator().manual_seed(L)
        how["starts"] = torch.stack([torch.randint(0, n + 3, (L,), generator=g) for n in lengths]).int()
    elif "starts" in how:
        how["starts"] = torch.tensor(how["starts"], dtype=torch.int32)
    if "slopes" in how:
        how["slopes"] = how["slopes"] * torch.arange(1, 7).float()
    _check_attend(_filled(k, v, lengths, "int8"), [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(lengths)], "int8", _queries(L, 3, 6, L, dtype), **how)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 3, 40])
def test_attend_ragged_batch(L, dtype):
    """Rows of their own lengths and counts of queries, one of them empty, one shorter than its queries."""
    lengths, counts = [300, 0, 64, 2, 129], [L, L, 0, L, max(L - 1, 1)]
    k, v = _rows(L, 5, 2, 300, dtype)
    c = _filled(k, v, lengths, "e4m3")
    rows = [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(lengths)]
    _check_attend(c, rows, "e4m3", _queries(L, 5, 8, L, dtype), counts=torch.tensor(counts, dtype=torch.int32))


@pytest.mark.parametrize("L", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_values_at_the_edges(dtype, L):
    """Scales far apart from block to block, blocks of zeros, large queries, infinities and NaN that were written and that queries do not see."""
    n = 400
    k, v = _rows(9, 1, 2, n, dtype)
    v[0, :, 64:128] *= 2.0 ** -9
    v[0, :, 128:192] = 0
    k[0, :, 192:256] *= 2.0 ** -12
    v[0, 1, 256:320] *= 2.0 ** 6
    k[0, 0, 330], v[0, 0, 340], v[0, 1, n - 1] = float("nan"), float("inf"), float("nan")
    c = _filled(k, v, [n], "int8")
    rows = [(k[0], v[0])]
    _check_attend(c, rows, "int8", _queries(1, 1, 8, L, dtype))
    q = _queries(2, 1, 8, L, dtype, size=50.0)
    q[0, 1] *= 2.0 ** -12
    q[0, 2] = 0
    _check_attend(c, rows, "int8", q)
    # a query that is not a number is its own affair
    bad = q.clone()
    bad[0, 3, 0, 5] = float("nan")
    out = c.attend(0, bad.to(DEV))
    good = c.attend(0, q.to(DEV))
    assert torch.isnan(out[0, 0, 3]).all()
    keep = torch.ones(L, 8, dtype=torch.bool)
    keep[0, 3] = False
    assert torch.equal(out[0, keep], good[0, keep])


def test_attend_query_strides():
    k, v = _rows(5, 2, 2, 150, torch.float16)
    c = _filled(k, v, [150, 150], "int8")
    for L in (1, 30):
        q = _queries(6, 2, 8, L, torch.float16).to(DEV)
        want = c.attend(0, q)
        assert torch.equal(c.attend(0, q.transpose(1, 2).contiguous().transpose(1, 2)), want)
        assert torch.equal(c.attend(0, q.transpose(2, 3).contiguous().transpose(2, 3)), want)
        assert torch.equal(c.attend(0, q[:, :, :1].expand(2, 8, L, 128)), c.attend(0, q[:, :, :1].repeat(1, 1, L, 1)))


# ------------------------------------------------------------------------------------------------ rows and pages
class _Rows:
    """A cache of several layers and what it should hold."""

    def __init__(self, lengths, H=2, layers=2, kind="int8", dtype=torch.float16, pages=None, max_tokens=600):
        self.kind, self.dtype, self.layers, self.H, self.seed = kind, dtype, layers, H, 100
        B = len(lengths)
        self.rows = [[(torch.zeros(H, 0, 128, dtype=dtype),) * 2 for _ in range(B)] for _ in range(layers)]
        self.c = _cache(B, H, max_tokens, layers=layers, kind=kind, dtype=dtype, pages=pages)
        self.grow(lengths)

    def grow(self, counts):
        T = max(counts)
        self.c.extend(counts)
        for layer in range(self.layers):
            self.seed += 1
            k, v = _rows(self.seed, len(counts), self.H, max(T, 1), self.dtype)
            self.c.write(layer, k[:, :, :T].to(DEV), v[:, :, :T].to(DEV))
            self.rows[layer] = [tuple(torch.cat([x, new[b, :, :counts[b]]], dim=1) for x, new in zip(row, (k, v)))
                                for b, row in enumerate(self.rows[layer])]

    def reorder(self, parents, on_device=False):
        self.c.reorder(torch.tensor(parents, device=DEV) if on_device else parents)
        self.rows = [[rows[b] for b in parents] for rows in self.rows]

    def truncate(self, lengths, rows=None):
        self.c.truncate(lengths, rows)
        for layer in range(self.layers):
            for b in range(self.c.batch) if rows is None else rows:
                n = lengths if isinstance(lengths, int) else int(lengths[b])
                self.rows[layer][b] = tuple(plain.cut(x, n, self.kind) for x in self.rows[layer][b])

    def check(self):
        for layer in range(self.layers):
            _holds(self.c, layer, self.rows[layer], self.kind)
        _pages_add_up(self.c)


@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [3, 2, 1, 0], [1, 1, 1, 1], [0, 0, 3, 3], [2, 0, 0, 1], [3, 3, 0, 0]])
def test_reorder(parents, on_device):
    r = _Rows([200, 64, 0, 130])
    r.reorder(parents, on_device)
    r.check()
    r.grow([70, 1, 64, 0])                       # rows that share pages go on apart
    r.check()
    r.reorder(parents, on_device)
    r.grow([1, 2, 3, 127])
    r.check()
    r.truncate(0)
    r.check()
    assert r.c.status.tolist()[0] == r.c.pages


@pytest.mark.parametrize("kind,dtype", [("int8", torch.float16), ("e4m3", torch.bfloat16)])
def test_truncate(kind, dtype):
    r = _Rows([200, 64, 129, 30], kind=kind, dtype=dtype)
    r.truncate([200, 63, 64, 10])
    r.check()
    r.grow([1, 1, 1, 100])
    r.check()
    r.truncate(70)
    r.check()
    r.truncate(65, rows=[0, 3])
    r.truncate(torch.tensor([65, 10, 500, 64], dtype=torch.int32, device=DEV))
    r.check()
    r.grow([64, 64, 64, 64])
    r.truncate(0, rows=[1, 2])
    r.check()
    r.grow([0, 300, 0, 3])
    r.check()


def test_a_shared_block_is_cut_for_one_row_only():
    r = _Rows([256, 10])
    r.reorder([0, 0])
    r.truncate(100, rows=[1])
    r.grow([5, 60])
    r.check()


def test_select_makes_another_batch_over_the_same_pages():
    r = _Rows([200, 64, 130])
    wide = r.c.select([0, 0, 2, 1, 2])
    assert wide.batch == 5
    for layer in range(r.layers):
        _holds(wide, layer, [r.rows[layer][b] for b in (0, 0, 2, 1, 2)], r.kind)
    _pages_add_up(r.c, wide)
    used = int((r.c.refs > 0).sum())
    r.c.free()
    _pages_add_up(r.c, wide)
    assert int((wide.refs > 0).sum()) == used
    k, v = _rows(8, 5, 2, 70, torch.float16)
    wide.extend(70)
    for layer in range(2):
        wide.write(layer, k.to(DEV), v.to(DEV))
        _holds(wide, layer, [tuple(torch.cat([x, y[i]], dim=1) for x, y in zip(r.rows[layer][b], (k, v))) for i, b in enumerate((0, 0, 2, 1, 2))], r.kind)
    narrow = wide.select(torch.tensor([4], device=DEV))
    with pytest.raises(ValueError, match="shared"):
        narrow.compacted()
    wide.release()
    _pages_add_up(narrow, wide)
    small = narrow.compacted()
    for layer in range(2):
        _holds(small, layer, [tuple(torch.cat([x, y[4]], dim=1) for x, y in zip(r.rows[layer][2], (k, v)))], r.kind)
    _pages_add_up(small)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_compaction(kind):
    r = _Rows([500, 130, 64, 300], kind=kind)
    r.reorder([0, 3, 2, 3])
    r.truncate(0, rows=[0])
    before, pages = r.c, int((r.c.refs > 0).sum())
    r.c = before.compacted()
    assert r.c.pages == pages and bool((r.c.refs > 0).all())
    r.check()
    with pytest.raises(ValueError, match="out of pages"):
        r.c.extend(64)
    r.c = r.c.compacted(pages=40)
    r.check()
    r.grow([100, 64, 300, 0])
    r.check()
    r.rows, r.c = r.rows, before                 # what it was copied from is as it was
    for layer in range(2):
        _holds(r.c, layer, [tuple(x[:, :n] for x, n in zip(row, [m] * 2)) for row, m in zip(r.rows[layer], (0, 300, 64, 300))], kind)


def test_freed_pages_come_again_lowest_first():
    r = _Rows([128, 128, 128], layers=1, pages=7)
    r.truncate(0, rows=[1])
    r.grow([0, 64, 64])
    assert r.c.table[r.c.slot.long()][:, :3].tolist() == [[0, 1, 0], [2, 3, 0], [4, 5, 3]]
    r.check()


def test_many_rows_and_long_tables():
    """1024 rows, a pool that is walked in many steps."""
    B = 1024
    c = _cache(B, 1, 200, pages=3000)
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 129, (B,), generator=g).tolist()
    k, v = _rows(2, B, 1, 128, torch.float16)
    c.append(k.to(DEV), v.to(DEV), counts)
    _holds(c, 0, [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(counts)], "int8")
    _pages_add_up(c)
    parents = torch.randint(0, B, (B,), generator=g).tolist()
    c.reorder(parents)
    _holds(c, 0, [(k[b, :, :counts[b]], v[b, :, :counts[b]]) for b in parents], "int8")
    _pages_add_up(c)


def test_pages_past_four_gigabytes():
    """Pages whose codes lie beyond 2^32 bytes: stored, read, attended, forked, cut and compacted."""
    H, far = 8, 65600                                         # 65600 pages of 8 heads: 2^32 bytes and a little more, keys and values each
    k, v = _rows(4, 2, H, 300, torch.float16)
    c = _cache(2, H, (far + 10) * 64, pages=far + 10)
    c.extend([far * 64, 0])                                   # (never written: what is looked at lies behind)
    c.append(k.to(DEV), v.to(DEV), [0, 300])
    assert int(c.table[c.slot[1], 0]) == far and far * H * 64 * 128 > 2 ** 32
    for L in (1, 20):
        q = _queries(L, 2, 16, L, torch.float16)
        nothing = torch.zeros(H, 0, 128, dtype=torch.float16)
        _check_attend(c, [(nothing, nothing), (k[1], v[1])], "int8", q, counts=torch.tensor([0, L], dtype=torch.int32))
    c.reorder([1, 1])
    _holds(c, 0, [(k[1], v[1])] * 2, "int8")
    c.truncate([300, 100])
    _holds(c, 0, [(k[1], v[1]), tuple(plain.cut(x[1], 100, "int8") for x in (k, v))], "int8")
    _pages_add_up(c)
    small = c.compacted()
    del c
    assert small.pages == 4
    _holds(small, 0, [(k[1], v[1]), tuple(plain.cut(x[1], 100, "int8") for x in (k, v))], "int8")


@pytest.mark.parametrize("window", [None, 200])
def test_attend_shares_of_many_rows(window):
    """More rows than a wavefront has lanes, whose blocks are shared out by their lengths, rows without tokens among them."""
    B = 150
    g = torch.Generator().manual_seed(2)
    lengths = [0 if b % 13 == 5 else int(n) for b, n in enumerate(torch.randint(1, 900, (B,), generator=g))]
    k, v = _rows(6, B, 1, max(lengths), torch.float16)
    c = _filled(k, v, lengths, "int8")
    q = _queries(3, B, 2, 1, torch.float16)
    _check_attend(c, [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(lengths)], "int8", q, **({} if window is None else {"window": window}))


# ------------------------------------------------------------------------------------------------ bounds, refusals, graphs
def test_room_is_checked_before_anything_is_launched():
    c = _cache(2, 1, 200, pages=4)
    c.extend([128, 127])
    with pytest.raises(ValueError, match="max_tokens"):
        c.extend(100)
    c.extend([0, 1])
    with pytest.raises(ValueError, match="out of pages"):
        c.extend(64)
    assert c.length.tolist() == [128, 128]
    c.extend(63)
    c.free([0])
    c.extend(torch.tensor([0, 1], dtype=torch.int32, device=DEV), bound=1)
    assert c.refresh() == [0, 192]
    # where a bound on the device's counts does not settle it, the counts do
    c.free()
    c.extend(torch.tensor([1, 190], dtype=torch.int32, device=DEV), bound=190)
    assert c.refresh() == [1, 190]
    c.extend(torch.tensor([190, 0], dtype=torch.int32, device=DEV), bound=190)         # 191 and 190 tokens: two full blocks each, all four pages
    with pytest.raises(ValueError, match="out of pages"):
        c.extend(torch.tensor([1, 0], dtype=torch.int32, device=DEV), bound=9)
    with pytest.raises(ValueError, match="max_tokens"):
        c.extend(torch.tensor([0, 11], dtype=torch.int32, device=DEV), bound=11)
    with pytest.raises(ValueError, match="bound=9"):
        c.extend(torch.tensor([0, 11], dtype=torch.int32, device=DEV), bound=9)


def test_what_the_device_refuses_changes_nothing():
    r = _Rows([100, 64], layers=1)
    r.c.reorder(torch.tensor([0, 2], device=DEV))
    with pytest.raises(RuntimeError, match="refused"):
        r.c.refresh()
    r.check()
    r.c.reorder(torch.tensor([-1, 0], device=DEV))
    with pytest.raises(RuntimeError, match="refused"):
        r.c.refresh()
    r.check()


@pytest.mark.parametrize("L", [1, 20])
def test_a_captured_step_goes_on_at_every_replay(L):
    """extend, write and attend in a graph: every replay stores and attends for the next tokens, and equals the same steps made eagerly, with
    eager work of the program between the replays; the replay that finds no room is refused and reported."""
    dtype, H, Hq, m = torch.bfloat16, 2, 8, 50
    k, v = _rows(7, 2, H, m, dtype)
    caches = [_filled(k, v, [m, m - 7], "int8", room=12 * L, pages=20) for _ in range(2)]
    ks, vs, q = (torch.zeros(2, n, L, 128, dtype=dtype, device=DEV) for n in (H, H, Hq))

    def step(c):
        c.extend(L)
        c.write(0, ks, vs)
        return c.attend(0, q, softcap=30.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _filled(k, v, [m, m - 7], "int8", room=100).attend(0, torch.zeros_like(q))       # (the first call on a stream sets things up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(10):
        kn, vn = _rows(50 + i, 2, H, L, dtype)
        ks.copy_(kn)
        vs.copy_(vn)
        q.copy_(_queries(i, 2, Hq, L, dtype))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step(caches[1])), i
        for x, y in zip(caches[0].read(0, m), caches[1].read(0, m)):
            assert torch.equal(x, y)
    assert caches[0].refresh() == caches[1].refresh()
    _pages_add_up(caches[0])


def test_a_replay_without_room_is_refused():
    k, v = _rows(7, 1, 1, 60, torch.float16)
    c = _filled(k, v, [60], "int8", pages=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(60)
    graph.replay()
    assert c.refresh() == [120]
    graph.replay()
    with pytest.raises(RuntimeError, match="refused"):
        c.refresh()
    assert c.refresh() == [120]


def test_numbers_from_the_host_in_a_graph():
    """Up to 512 rows they are part of the launch and the same at every replay; beyond that the host's memory would be read again, which is refused."""
    r = _Rows([200, 64, 130], layers=1)
    k, v = (x.to(DEV) for x in _rows(90, 3, 2, 70, torch.float16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.c.reorder([0, 0, 1])
        r.c.truncate([100, 1000, 3])
        r.c.extend([1, 70, 64])
        r.c.write(0, k, v)
    junk = [torch.full((1 << 16,), i, pin_memory=True) for i in range(4)]       # (what pinned memory was about would be overwritten)
    for _ in range(3):
        graph.replay()
        rows = [r.rows[0][b] for b in (0, 0, 1)]
        rows = [tuple(plain.cut(x, n, r.kind) for x in row) for row, n in zip(rows, (100, 1000, 3))]
        r.rows[0] = [tuple(torch.cat([x, y[b, :, :n].cpu()], dim=1) for x, y in zip(row, (k, v))) for b, (row, n) in enumerate(zip(rows, (1, 70, 64)))]
        assert r.c.refresh() == [x[0].shape[1] for x in r.rows[0]]
        r.check()
    assert len(junk) == 4
    wide = _cache(600, 1, 70)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=DEV)
        for call in (lambda: wide.reorder([0] * 600), lambda: wide.truncate([3] * 600), lambda: wide.extend([1] * 600)):
            with pytest.raises(RuntimeError, match="captured"):
                call()


def test_another_stream():
    k, v = _rows(11, 1, 2, 300, torch.float16)
    q = _queries(1, 1, 8, 1, torch.float16).to(DEV)
    want = _filled(k, v, [300], "int8").attend(0, q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _filled(k, v, [300], "int8").attend(0, q)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_tokens_are_stored_once_a_layer_and_extend():
    k, v = _rows(1, 1, 1, 70, torch.float16)
    k, v = k.to(DEV), v.to(DEV)
    c = _cache(1, 1, 300)
    c.extend(70)
    with pytest.raises(ValueError, match="70"):
        c.write(0, k[:, :, :69], v[:, :, :69])
    c.write(0, k, v)
    for args in ((k, v), (k.transpose(2, 3).contiguous().transpose(2, 3), v)):
        with pytest.raises(ValueError, match="already"):
            c.write(0, *args)
    c.extend(torch.tensor([3], device=DEV), bound=5)
    with pytest.raises(ValueError, match="5"):
        c.write(0, k[:, :, :4], v[:, :, :4])
    c.write(0, k[:, :, :6], v[:, :, :6])
    _holds(c, 0, [tuple(torch.cat([x, x[:, :, :3]], dim=2)[0].cpu() for x in (k, v))], "int8")


@pytest.mark.parametrize("L", [1, 3, 20])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["freed", "cut"])
def test_what_a_tail_held_before_decides_nothing(how, dtype, L):
    """Tokens behind a row's end, as large as the type has them, beside small ones in the same tail."""
    big = torch.finfo(dtype).max / 4
    k, v = _rows(2, 1, 2, 40, dtype)
    k, v = k * 2.0 ** -6, v * 2.0 ** -8                       # (fp16: v from 2^-24 on, of which a factor of 2^-9 would leave nothing)
    old = torch.full((1, 2, 60, 128), big, dtype=dtype)
    c = _cache(1, 2, 300, dtype=dtype)
    if how == "freed":
        c.append(old.to(DEV), old.to(DEV))
        c.free()
    else:
        c.append(k[:, :, :7].to(DEV), v[:, :, :7].to(DEV))
        c.append(old[:, :, :50].to(DEV), old[:, :, :50].to(DEV))
        c.truncate(7)
    have = c.length.tolist()[0]
    c.append(k[:, :, have:21].to(DEV), v[:, :, have:21].to(DEV))
    _check_attend(c, [(k[0, :, :21], v[0, :, :21])], "int8", _queries(1, 1, 8, L, dtype, 60.0))


def test_tokens_of_rows_that_have_moved_are_not_stored():
    k, v = _rows(1, 2, 1, 10, torch.float16)
    k, v = k.to(DEV), v.to(DEV)
    c = _cache(2, 1, 300)
    for move in (lambda: c.reorder([1, 0]), lambda: c.truncate(3), lambda: c.free([1])):
        c.free()
        c.extend(10)
        move()
        with pytest.raises(ValueError, match="moved or cut"):
            c.write(0, k, v)
    c.extend(10)
    new = c.select([0])
    with pytest.raises(ValueError, match="moved or cut"):
        new.write(0, k[:1], v[:1])
    c.write(0, k, v)                                          # (the batch that was copied has not moved)


def test_numbers_past_32_bits_stop_at_their_end():
    k, v = _rows(3, 2, 1, 100, torch.float16)
    c = _filled(k, v, [100, 100], "int8", room=50)
    q = _queries(1, 2, 4, 3, torch.float16).to(DEV)
    far = 2 ** 32 + 5
    none, lse = c.attend(0, q, starts=torch.tensor([far, far], device=DEV), return_lse=True)
    assert not none.any() and bool((lse == float("-inf")).all())
    everything = c.attend(0, q, prefix=torch.tensor([100, 100], device=DEV))
    assert torch.equal(c.attend(0, q, prefix=torch.tensor([far, far], device=DEV)), everything)
    c.truncate(2 ** 32)
    c.truncate(torch.tensor([far, far], device=DEV))
    c.extend(torch.tensor([1, 2], device=DEV), bound=far)
    assert c.refresh() == [101, 102]


def test_beams_of_one_length_need_no_reading_back():
    """Parents that only the device knows leave the host's bounds as they are where all rows are alike."""
    k, v = _rows(1, 4, 1, 64, torch.float16)
    c = _filled(k, v, [64] * 4, "int8", pages=9)
    c.refresh = lambda: pytest.fail("read back")
    for step in range(64):
        c.reorder(torch.tensor([step % 4, 0, 1, 1], device=DEV))
        c.extend(1)
        c.write(0, k[:, :, :1].to(DEV), v[:, :, :1].to(DEV))
    assert c.length.tolist() == [128] * 4
    _pages_add_up(c)


def test_refusals():
    c = _cache(2, 2, 200, layers=2)
    x = torch.zeros(2, 2, 5, 128, dtype=torch.float16, device=DEV)
    q = torch.zeros(2, 8, 1, 128, dtype=torch.float16, device=DEV)
    bad = [lambda: c.extend(-1), lambda: c.extend([1]), lambda: c.extend([1, -2]), lambda: c.extend(torch.ones(2, dtype=torch.int32, device=DEV)),
           lambda: c.extend(torch.ones(3, dtype=torch.int32, device=DEV), bound=3), lambda: c.extend([1, 4], bound=3),
           lambda: c.extend(torch.ones(2, device=DEV), bound=3),
           lambda: c.append(x, x), lambda: c.write(2, x, x), lambda: c.write(-1, x, x), lambda: c.write(0, x[:1], x[:1]), lambda: c.write(0, x, x[:, :, :4]),
           lambda: c.write(0, x.bfloat16(), x.bfloat16()), lambda: c.write(0, x[..., :64], x[..., :64]),
           lambda: c.reorder([0]), lambda: c.reorder([0, 2]), lambda: c.reorder([0, -1]), lambda: c.reorder(torch.zeros(2, device=DEV)), lambda: c.select([]),
           lambda: c.select([5]), lambda: c.truncate(-1), lambda: c.truncate([1]), lambda: c.truncate([1, -1]), lambda: c.truncate(1, rows=[2]), lambda: c.free([-1]),
           lambda: c.read(2), lambda: c.read(0, -1), lambda: c.read(0, 3, dtype=torch.int32),
           lambda: c.attend(2, q), lambda: c.attend(0, q[:1]), lambda: c.attend(0, q[:, :7]), lambda: c.attend(0, q.bfloat16()), lambda: c.attend(0, q.float()),
           lambda: c.attend(0, q.repeat(1, 3, 1, 1)), lambda: c.attend(0, q, softcap=0.0), lambda: c.attend(0, q, softcap=-1.0), lambda: c.attend(0, q, window=0),
           lambda: c.attend(0, q, slopes=torch.zeros(4, device=DEV)), lambda: c.attend(0, q, prefix=torch.zeros(2, device=DEV)),
           lambda: c.attend(0, q, prefix=[1, 2]), lambda: c.attend(0, q, starts=torch.zeros(2, 2, dtype=torch.int32, device=DEV)),
           lambda: c.attend(0, q, starts=torch.zeros(2, dtype=torch.int32)), lambda: c.compacted(pages=0),
           lambda: _cache(0, 1, 10), lambda: _cache(1025, 1, 10), lambda: _cache(1, 1, 10, kind="int4"), lambda: _cache(1, 1, 10, dtype=torch.float32),
           lambda: _cache(1, 1, 10, head_dim=64), lambda: _cache(1, 0, 10), lambda: _cache(1, 1, 0), lambda: _cache(1, 1, 10, pages=-1)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    for call in (lambda: c.write(0, x.cpu(), x.cpu()), lambda: c.attend(0, q.cpu()), lambda: _cache(1, 1, 10, device="cpu")):
        with pytest.raises(RuntimeError):
            call()
    assert c.refresh() == [0, 0]
