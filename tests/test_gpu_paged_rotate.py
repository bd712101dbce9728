"""GPU: keys that are turned by their positions on their way into the paged 8-bit cache, and the queries beside them, against the definition: bit for bit, and
against angles in 64 bits."""
import pytest
import torch

import paged_rows as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def _tables(positions, turned, theta=10000.0):
    half = turned // 2
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


def _turned(x, cos, sin, interleaved, key=False):
    """x [..., T, 128] in 16 bits by cos, sin [T, R / 2]: two products and their sum, each rounded to 32 bits, then once to 16."""
    half = cos.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a.float(), b.float()
    u, v = a * cos - b * sin, b * cos + a * sin
    if key:
        u, v = plain.finite(u), plain.finite(v)
        u, v = (plain.to_type(t.double(), x.dtype) for t in (u, v))
    out = x.clone()
    if key:
        out = plain.finite(out)
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = u.to(x.dtype), v.to(x.dtype)
    else:
        out[..., :half], out[..., half:2 * half] = u.to(x.dtype), v.to(x.dtype)
    return out


def _cache(*args, **kw):
    from kvquant import PagedKVCache
    return PagedKVCache(*args, **kw)


def _random(seed, *shape, dtype, scale=2.0):
    return (torch.randn(*shape, 128, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _holds(c, layer, rows, kind):
    n = max([k.shape[1] for k, _ in rows] + [1])
    got_k, got_v = c.read(layer, n, dtype=torch.float32)
    assert c.length.tolist() == [k.shape[1] for k, _ in rows]
    for b, (k, v) in enumerate(rows):
        for got, x in ((got_k, k), (got_v, v)):
            assert torch.equal(got[b, :, :x.shape[1]].cpu().double(), plain.held(x, kind)), (b, layer)
            assert not got[b, :, x.shape[1]:].any()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("turned,interleaved", [(128, False), (128, True), (64, False), (48, True), (16, False)])
def test_turned_and_stored(turned, interleaved, dtype, kind):
    """Ragged rows whose tokens arrive in pieces: the queries' and the stored keys' bits are the definition's, the values are as they come."""
    B, H, Hq = 3, 2, 6
    counts = [[70, 1, 0], [1, 1, 1], [0, 63, 5], [130, 64, 62]]
    total = [sum(c[b] for c in counts) for b in range(B)]
    k, v, q = (_random(s, B, h, max(total), dtype=dtype) for s, h in ((1, H), (2, H), (3, Hq)))
    cos, sin = _tables(max(total), turned)
    c = _cache(B, H, max(total), kind=kind, dtype=dtype)
    at = [0] * B
    for step in counts:
        T = max(step) + 2
        ks, vs, qs = (torch.full((B, h, T, 128), float("nan"), dtype=dtype) for h in (H, H, Hq))
        for b, n in enumerate(step):
            for to, x in ((ks, k), (vs, v), (qs, q)):
                to[b, :, :n] = x[b, :, at[b]:at[b] + n]
        c.extend(step)
        got, got_k = c.write_rotated(0, qs.to(DEV), ks.to(DEV), vs.to(DEV), cos.to(DEV), sin.to(DEV), interleaved=interleaved, return_keys=True)
        assert got.shape == qs.shape and got_k.shape == ks.shape and got.dtype == dtype
        for b, n in enumerate(step):
            here = slice(at[b], at[b] + n)
            want = _turned(q[b, :, here], cos[here], sin[here], interleaved)
            assert torch.equal(got[b, :, :n].cpu(), want)
            assert torch.equal(got_k[b, :, :n].cpu(), _turned(k[b, :, here], cos[here], sin[here], interleaved, key=True))
            assert not got[b, :, n:].any() and not got_k[b, :, n:].any()
            # the formula in 64 bits: half a step of the type, and of 32 bits the products' and the sum's
            exact = _turned(q[b, :, here].double(), cos[here].double(), sin[here].double(), interleaved) if n else want.double()
            size = q[b, :, here].double().abs().amax() if n else 0.0
            eps = torch.finfo(dtype).eps / 2
            assert bool(((want.double() - exact).abs() <= exact.abs() * eps * (1 + eps) + 4 * 2.0 ** -24 * size + torch.finfo(dtype).smallest_normal * eps).all())
        at = [a + n for a, n in zip(at, step)]
    _holds(c, 0, [(_turned(k[b, :, :n], cos[:n], sin[:n], interleaved, key=True), v[b, :, :n]) for b, n in enumerate(total)], kind)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_rows_with_strides(dtype):
    """Packed prompts, one of them empty, as slices of one projection: the same bytes as each row by itself, and tokens behind the last row are 0."""
    lengths, H, Hq = [0, 130, 1, 64, 300, 0], 3, 9
    N = sum(lengths)
    wide = torch.randn(N + 5, (Hq + 2 * H) * 128, generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    q, k, v = (x.view(1, N + 5, -1, 128).transpose(1, 2) for x in wide.split([Hq * 128, H * 128, H * 128], dim=1))
    cos, sin = _tables(400, 128)
    offsets = torch.tensor([0, 0, 130, 131, 195, 495, 495], dtype=torch.int32, device=DEV)
    for wait in (0, 2):                                                     # into empty rows, and behind what is there
        packed, single = (_cache(6, H, 700, dtype=dtype) for _ in range(2))
        if wait:
            first = _random(5, 6, H, 100, dtype=dtype).to(DEV)
            for c in (packed, single):
                c.append(first, first, [3, 64, 0, 100, 7, 1])
        before = single.length.tolist()
        packed.extend(lengths)
        turned, keys = packed.write_rotated(0, q, k, v, cos.to(DEV), sin.to(DEV), offsets=offsets, return_keys=True)
        assert turned.shape == (1, Hq, N + 5, 128) and not turned[:, :, N:].any() and not keys[:, :, N:].any()
        at = 0
        for b, n in enumerate(lengths):
            place = slice(before[b], before[b] + n)
            want = _turned(q[0, :, at:at + n].cpu(), cos[place], sin[place], False)
            assert torch.equal(turned[0, :, at:at + n].cpu(), want)
            at += n
        single.extend(lengths)
        T = max(lengths)
        ks, vs = (torch.zeros(6, H, T, 128, dtype=dtype, device=DEV) for _ in range(2))
        at = 0
        for b, n in enumerate(lengths):
            ks[b, :, :n], vs[b, :, :n] = k[0, :, at:at + n], v[0, :, at:at + n]
            at += n
        assert single.write_rotated(0, None, ks, vs, cos.to(DEV), sin.to(DEV)) is None
        for x, y in zip(packed.read(0, 500), single.read(0, 500)):
            assert torch.equal(x, y)
        assert packed.refresh() == single.refresh()


def test_positions_and_starts():
    """Padding in front stands at 0, positions of the caller's own are taken as they are, packed ones as well."""
    B, H, T = 3, 2, 90
    k, v, q = (_random(s, B, h, T, dtype=torch.bfloat16) for s, h in ((1, H), (2, H), (3, 4)))
    cos, sin = _tables(1000, 128)
    starts = torch.tensor([0, 17, 89], dtype=torch.int32)
    at = (torch.arange(T) - starts[:, None]).clamp(min=0)
    own = torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(9))
    for given, place in ((dict(starts=starts.to(DEV)), at), (dict(positions=own.to(DEV)), own), (dict(positions=own.to(torch.int32).t().contiguous().t().to(DEV)), own)):
        c = _cache(B, H, 200, dtype=torch.bfloat16)
        c.extend(T)
        got = c.write_rotated(0, q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), **given)
        want = torch.stack([_turned(q[b], cos[place[b]], sin[place[b]], False) for b in range(B)])
        assert torch.equal(got.cpu(), want)
        _holds(c, 0, [(_turned(k[b], cos[place[b]], sin[place[b]], False, key=True), v[b]) for b in range(B)], "int8")
        c.refresh()
    c = _cache(2, H, 200, dtype=torch.bfloat16)
    c.extend([60, 30])
    offsets = torch.tensor([0, 60, 90], dtype=torch.int64, device=DEV)
    got = c.write_rotated(0, q[:1].to(DEV), k[:1].to(DEV), v[:1].to(DEV), cos.to(DEV), sin.to(DEV), offsets=offsets, positions=own[:1].to(DEV))
    assert torch.equal(got.cpu(), _turned(q[:1], cos[own[0]], sin[own[0]], False))
    c.refresh()


def test_what_the_device_alone_can_see():
    """Positions behind the table count as its nearest and are told; offsets that do not fit leave their rows as they were, in or out of range."""
    H, T = 2, 40
    k, v, q = (_random(s, 1, h, T, dtype=torch.float16).to(DEV) for s, h in ((1, H), (2, H), (3, 4)))
    cos, sin = (t.to(DEV) for t in _tables(50, 128))
    c = _cache(1, H, 200, dtype=torch.float16)
    c.extend(T)
    own = torch.arange(T, device=DEV).view(1, T) - 3
    own[0, -1] = 2 ** 31 - 1
    got = c.write_rotated(0, q, k, v, cos, sin, positions=own)
    near = own[0].clamp(0, 49).cpu()
    assert torch.equal(got.cpu(), _turned(q.cpu(), cos.cpu()[near], sin.cpu()[near], False))
    with pytest.raises(RuntimeError, match="refused on the device"):
        c.refresh()
    for bad in ([0, 20, 41], [-1, 19, 40], [0, 21, 40], [0, 20, 2 ** 31 - 1], [30, 20, 40], [2 ** 31 - 1, -2 ** 31, 40]):
        c = _cache(2, H, 200, dtype=torch.float16)
        c.extend(20)
        got, keys = c.write_rotated(0, q, k, v, cos, sin, offsets=torch.tensor(bad, dtype=torch.int32, device=DEV), return_keys=True)
        stored, _ = c.read(0, 20)
        for b in range(2):
            if bad[b] >= 0 and bad[b + 1] <= 40 and bad[b + 1] - bad[b] == 20:
                assert torch.equal(stored[b].cpu(), _turned(k[0, :, bad[b]:bad[b + 1]].cpu(), cos.cpu()[:20], sin.cpu()[:20], False, key=True))
            else:
                assert not stored[b].any()
        with pytest.raises(RuntimeError, match="refused on the device"):
            c.refresh()


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_edges(dtype):
    """Infinities, NaN and keys whose turned pair passes the type's end."""
    H, T = 1, 70
    k, v, q = (_random(s, 1, h, T, dtype=dtype) for s, h in ((1, H), (2, H), (3, 2)))
    for x in (k, v, q):
        x[0, 0, 3, 5], x[0, 0, 4, 70], x[0, 0, 66, 0], x[0, 0, 69, 127] = float("inf"), float("nan"), float("-inf"), float("nan")
    k[0, 0, 10] = torch.finfo(dtype).max
    k[0, 0, 67] = -torch.finfo(dtype).max
    cos, sin = _tables(T, 96)
    c = _cache(1, H, T, dtype=dtype)
    c.extend(T)
    got = c.write_rotated(0, q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV))
    assert torch.equal(got.cpu().nan_to_num(nan=77.0), _turned(q, cos, sin, False).nan_to_num(nan=77.0))
    _holds(c, 0, [(_turned(k[0], cos, sin, False, key=True), v[0])], "int8")


def test_many_rows_and_tokens():
    """More rows than the native bookkeeping takes from the host, one token each; and a prompt of many blocks by several heads a workgroup."""
    cos, sin = _tables(5000, 128)
    k, v, q = (_random(s, 700, h, 1, dtype=torch.float16) for s, h in ((1, 1), (2, 1), (3, 8)))
    c = _cache(700, 1, 10)
    c.extend(1)
    got = c.write_rotated(0, q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV))
    assert torch.equal(got.cpu(), _turned(q, cos[:1], sin[:1], False))
    c.extend(1)
    got = c.write_rotated(0, q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV))
    assert torch.equal(got.cpu(), _turned(q, cos[1:2], sin[1:2], False))
    n = 4999
    k, v, q = (_random(s, 1, h, n, dtype=torch.bfloat16) for s, h in ((1, 4), (2, 4), (3, 28)))
    c = _cache(1, 4, n, dtype=torch.bfloat16)
    c.extend(n)
    got = c.write_rotated(0, q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), interleaved=True)
    assert torch.equal(got.cpu(), _turned(q, cos[:n], sin[:n], True))
    _holds(c, 0, [(_turned(k[0], cos[:n], sin[:n], True, key=True), v[0])], "int8")


def test_a_captured_step_goes_on():
    """extend, write_rotated and attend in one graph: every replay is the eager step, with work on other rows in between."""
    H, Hq, n, steps = 2, 8, 62, 5
    k, v, q = (_random(s, 2, h, n + steps, dtype=torch.bfloat16).to(DEV) for s, h in ((1, H), (2, H), (3, Hq)))
    cos, sin = (t.to(DEV) for t in _tables(n + steps + 3, 128))
    eager, captured = (_cache(2, H, n + steps + 1, dtype=torch.bfloat16) for _ in range(2))
    for c in (eager, captured):
        c.extend(n)
        c.write_rotated(0, None, k[:, :, :n], v[:, :, :n], cos, sin)
    qs, ks, vs = (x[:, :, n:n + 1].clone() for x in (q, k, v))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.extend(1)
        turned = captured.write_rotated(0, qs, ks, vs, cos, sin)
        out = captured.attend(0, turned)
    for i in range(steps):
        for to, x in ((qs, q), (ks, k), (vs, v)):
            to.copy_(x[:, :, n + i:n + i + 1])
        graph.replay()
        eager.extend(1)
        want_q = eager.write_rotated(0, q[:, :, n + i:n + i + 1], k[:, :, n + i:n + i + 1], v[:, :, n + i:n + i + 1], cos, sin)
        want = eager.attend(0, want_q, longest=n + steps + 1)
        torch.cuda.synchronize()
        assert torch.equal(turned, want_q) and torch.equal(out, want), i
    assert captured.refresh() == [n + steps] * 2
    for x, y in zip(captured.read(0), eager.read(0)):
        assert torch.equal(x, y)


def test_another_stream():
    H, T = 2, 200
    k, v, q = (_random(s, 1, h, T, dtype=torch.float16).to(DEV) for s, h in ((1, H), (2, H), (3, 4)))
    cos, sin = (t.to(DEV) for t in _tables(T, 128))
    c = _cache(1, H, T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.extend(T)
        got = c.write_rotated(0, q, k, v, cos, sin)
    side.synchronize()
    assert torch.equal(got.cpu(), _turned(q.cpu(), cos.cpu(), sin.cpu(), False))


def test_refusals():
    H, T = 2, 10
    k, v, q = (_random(s, 2, h, T, dtype=torch.float16).to(DEV) for s, h in ((1, H), (2, H), (3, 4)))
    cos, sin = (t.to(DEV) for t in _tables(64, 128))
    c = _cache(2, H, 64, layers=2)
    c.extend(T)
    i32 = dict(dtype=torch.int32, device=DEV)
    for args, kw, says in (((2, q, k, v, cos, sin), {}, "layer 2"), ((0, q, k[:1], v, cos, sin), {}, "keys must be"), ((0, q[..., :64], k, v, cos, sin), {}, "queries must be"),
                           ((0, q[:, :, :5], k, v, cos, sin), {}, "a row"), ((0, q[:, :, :5], k[:, :, :5], v[:, :, :5], cos, sin), {}, "grown"),
                           ((0, q.bfloat16(), k, v, cos, sin), {}, "must be torch.float16"), ((0, q, k, v, cos.half(), sin.half()), {}, "float32"),
                           ((0, q, k, v, cos, sin[:5]), {}, "sine"), ((0, q, k, v, cos[:, :12], sin[:, :12]), {}, "multiple of 16"),
                           ((0, q, k, v, cos[:9], sin[:9]), {}, "9 positions"), ((0, q, k, v, cos, sin), dict(offsets=torch.zeros(2, **i32)), "keys must be"),
                           ((0, q, k, v, cos, sin), dict(starts=torch.zeros(3, **i32)), "starts"), ((0, q, k, v, cos, sin), dict(positions=torch.zeros(2, 9, **i32)), "positions"),
                           ((0, q, k, v, cos, sin), dict(positions=torch.zeros(2, T, device=DEV)), "whole numbers"),
                           ((0, q, k, v, cos, sin), dict(positions=torch.zeros(2, T, **i32), starts=torch.zeros(2, **i32)), "twice"),
                           ((0, q[:0].reshape(2, 0, T, 128), k, v, cos, sin), {}, "0 query heads")):
        with pytest.raises(ValueError, match=says):
            c.write_rotated(*args, **kw)
    with pytest.raises(ValueError, match="offsets"):
        c.write_rotated(0, q[:1], k[:1], v[:1], cos, sin, offsets=torch.zeros(2, **i32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.write_rotated(0, q, k, v, cos.cpu(), sin.cpu())
    with pytest.raises(RuntimeError, match="no gradients"):
        c.write_rotated(0, q.clone().requires_grad_(), k, v, cos, sin)
    c.write_rotated(0, q, k, v, cos, sin)
    with pytest.raises(ValueError, match="has stored"):
        c.write_rotated(0, q, k, v, cos, sin)
    with pytest.raises(ValueError, match="layer 1 has not stored"):
        c.attend(1, q)
    c.write(1, k, v)                                                        # a layer without positions beside one with them
    assert c.refresh() == [T, T]


def test_what_would_be_recorded_is_refused():
    """Gradients while they are recorded, tangents with and without: of tokens and of tables, each by itself, by the native call and (with positions) by the other; nothing is stored then."""
    from torch.autograd import forward_ad
    H, T = 2, 10
    given = [*(_random(s, 2, h, T, dtype=torch.float16).to(DEV) for s, h in ((1, 4), (2, H), (3, H))), *(t.to(DEV) for t in _tables(64, 128))]
    c = _cache(2, H, 64)
    c.extend(T)
    where = torch.arange(T, dtype=torch.int32, device=DEV).expand(2, T).contiguous()
    for how in (dict(), dict(positions=where)):
        for i in range(5):
            args = list(given)
            args[i] = args[i].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradients"):
                c.write_rotated(0, *args, **how)
            with forward_ad.dual_level(), torch.no_grad():
                args[i] = forward_ad.make_dual(given[i].clone(), torch.ones_like(given[i]))
                with pytest.raises(RuntimeError, match="no tangents"):
                    c.write_rotated(0, *args, **how)
    learned = [*given[:3], *(t.clone().requires_grad_() for t in given[3:])]
    with torch.no_grad():                                                                    # learned tables, at inference
        got = c.write_rotated(0, *learned)
    assert torch.equal(got, _turned(given[0].cpu(), given[3][:T].cpu(), given[4][:T].cpu(), False).to(DEV))


def test_tables_that_lie_anywhere():
    """Tables off 16 bytes, transposed, and as every other row of a larger one: the same bits."""
    q, k, v = (_random(s, 2, h, 70, dtype=torch.float16).to(DEV) for s, h in ((31, 4), (32, 2), (33, 2)))
    cos, sin = (t.to(DEV) for t in _tables(80, 64))
    want = None
    for lay in (lambda t: t, lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].view(80, 32), lambda t: t.t().contiguous().t(), lambda t: t.repeat_interleave(2, dim=0)[::2]):
        c = _cache(2, 2, 80)
        c.extend(70)
        got = (*c.write_rotated(0, q, k, v, lay(cos), lay(sin), return_keys=True), *c.read(0, 70))
        want = got if want is None else want
        assert all(torch.equal(a, b) for a, b in zip(got, want))
