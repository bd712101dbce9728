"""GPU: attention over the paged 8-bit cache where blocks, or tokens of a tail, are of very different size: a query's result is made of the tokens that it sees, whatever
else lies in the row, and small values count beside large ones that weigh nothing."""
import pytest
import torch

import paged_rows as plain
from test_gpu_paged_cache import DEV, DTYPES, _cache, _filled, _queries, _rows

pytestmark = pytest.mark.gpu
# how far values (and, in a tail, keys) that nobody sees are from the others: powers of two that leave the type's range alone
FAR = {torch.float16: (-12, 12), torch.bfloat16: (-60, 60)}


def _blocks_largest(v, kind):
    """The largest |value| of a token's full block, or of the token itself in the tail, [H, n, 1]."""
    n, full = v.shape[1], v.shape[1] // 64 * 64
    own = v.abs().amax(dim=-1, keepdim=True)
    own[:, :full] = own[:, :full].view(v.shape[0], -1, 64, 1).amax(dim=2).repeat_interleave(64, dim=1)
    return own


def _check(out, lse, q, k, v, kind, **how):
    """One row's out [L, Hq, 128] and lse [Hq, L] against the definition, with a bound made of what a query sees:
    scores and their sum as in paged_rows.attend; weights rounded to fp16 (2^-11 of themselves); those below its normal numbers are off by 2^-25 at most, in
    a unit in which the largest P_j s_j is 2^8, and 2^6 in a block of e4m3 codes (s_j: what a code of one stands for, V_j / 127, V_j / 448, or in the tail V_j / 64 at most, V_j
    the largest value of the block or the tail's token), times codes of at most 127, 448 and 128: the worst is a code of 448 beside a largest P_j V_j in the tail,
    2^-25 * 448 * 2^-8 / 64 = 3.5 * 2^-32 of it, for every token.  A tail's values, in fp16 with their token's largest at 64 or more, are off by 2^-24 of that unit at the
    most, 2^-30 of P_j V_j."""
    dtype, L, m = q.dtype, q.shape[1], k.shape[1]
    held_k, held_v = plain.held(k, kind), plain.held(v, kind)
    want, wl, _, tl = plain.attend(q, held_k, held_v, **how)
    mass = plain.attend(q, held_k, held_v.abs(), **how)[0]
    large = plain.attend(q, held_k, _blocks_largest(held_v, kind).expand_as(held_v), **how)[0]
    tol = (2 * tl.T[..., None] + 2.0 ** -11 + 2 * m * 2.0 ** -24) * mass + (3.5 * m + 4) * 2.0 ** -32 * 1.01 * large
    bound = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    got, gl = out.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isinf(gl), torch.isinf(wl)) and torch.isfinite(got).all()
    ok = torch.isfinite(wl)
    assert ((gl - wl).abs()[ok] <= tl[ok] + 2.0 ** -23 * wl.abs()[ok]).all()
    off = (got - want).abs() / bound
    assert (off <= 1).all(), (float(off.max()), float((got - want).norm() / want.norm()))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("L", [2, 4, 17, 40, 130])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [0, 1])
def test_values_of_another_document_change_nothing(up, dtype, L, kind):
    """Two documents, the second from a block's start on, queries of both: the first one's values, and keys, as they are and by a power of two smaller or larger: the
    second one's results are the same bits, and those of the definition."""
    n, at = 300 + L, 128
    k, v = _rows(L, 1, 2, n, dtype)
    v = v * 2.0 ** (-4 if up else 0)
    q = _queries(L, 1, 8, L, dtype)
    starts = torch.tensor([[0] * (L // 2) + [at] * (L - L // 2)], dtype=torch.int32)
    got = []
    for by in (0, FAR[dtype][up]):
        w, x = v.clone(), k.clone()
        w[:, :, :at] *= 2.0 ** by
        x[:, :, :at] *= 2.0 ** (by / 4)
        got.append(_filled(x, w, [n], kind).attend(0, q.to(DEV), starts=starts.to(DEV), return_lse=True))
    (out, lse), (out1, lse1) = got
    assert torch.equal(out[:, L // 2:], out1[:, L // 2:]) and torch.equal(lse[..., L // 2:], lse1[..., L // 2:])
    v[:, :, :at] = 0                                          # (the second document's queries do not see them: what the bound is made of)
    _check(out1[0, L // 2:], lse1[0, :, L // 2:], q[0, :, L // 2:], k[0], v[0], kind, starts=torch.tensor(at))


@pytest.mark.parametrize("L", [3, 17, 40])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far", [-1, 1])
def test_tokens_of_a_tail_that_others_see_change_nothing(far, dtype, L):
    """A tail whose tokens belong to two documents, and one whose newest tokens only the newest queries see: keys and values of either, larger or smaller."""
    n, at = 64 * 3 + 30, 64 * 3 + 20
    k, v = _rows(L, 1, 2, n, dtype)
    k, v = k * 2.0 ** -2, v * 2.0 ** -2
    by = 2.0 ** (far * FAR[dtype][1])
    q = _queries(L, 1, 8, L, dtype)
    for where, mine in ((slice(64 * 3, at), dict(starts=torch.tensor([at], dtype=torch.int32))), (slice(n - 1, n), {})):
        got = []
        for scale in (1.0, by):
            x, w = k.clone(), v.clone()
            x[:, :, where] *= scale
            w[:, :, where] *= scale
            got.append(_filled(x, w, [n], "int8").attend(0, q.to(DEV), return_lse=True, **{name: t.to(DEV) for name, t in mine.items()}))
        last = L if mine else L - 1                           # (the newest query sees the newest token)
        assert torch.equal(got[0][0][:, :last], got[1][0][:, :last]) and torch.equal(got[0][1][..., :last], got[1][1][..., :last])
        if mine:
            w = v.clone()
            w[:, :, :at] = 0
            _check(got[1][0][0], got[1][1][0], q[0], k[0], w[0], "int8", starts=torch.tensor(at))


def _attend(k, v, q, kind):
    """out [L, Hq, 128] and lse [Hq, L] of one row; for a few queries among 63 more rows, so that a wavefront takes several of its blocks."""
    n, H, L = k.shape[2], k.shape[1], q.shape[2]
    if L > 3:
        out, lse = _filled(k, v, [n], kind).attend(0, q.to(DEV), return_lse=True)
    else:
        c = _cache(64, H, n + 10, pages=n // 64 + 64, kind=kind, dtype=k.dtype)
        c.append(*(x.to(DEV).expand(64, H, n, 128) for x in (k, v)), [n] + [5] * 63)
        out, lse = c.attend(0, q.to(DEV).expand(64, -1, L, 128), return_lse=True)
    return out[0], lse[0]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("L", [1, 3, 40, 130])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["large ones weigh nothing", "small ones weigh most", "as they come"])
@pytest.mark.parametrize("where", ["page", "tail"])
def test_small_values_beside_large_ones(where, what, dtype, L, kind):
    """One block (or the tail) of values larger than the others by far: with weights of e^-200, which leaves the others' values alone; with weights a thousandth of the
    others', whose sum counts; and as the scores come."""
    n = 650
    small, large = (-80, 40) if dtype == torch.bfloat16 else (-13, 9)
    k, v = _rows(L, 1, 8, n, dtype)
    far = slice(64, 128) if where == "page" else slice(640, 650)
    k[..., 0] = 0
    q = _queries(L, 1, 8, L, dtype)
    q[..., 0] = 40
    if what != "as they come":
        k[:, :, far, 0] = -60 if what == "large ones weigh nothing" else -2
    v = v.float() * 2.0 ** small
    v[:, :, far] *= 2.0 ** (large - small)
    v = v.to(dtype)
    out, lse = _attend(k, v, q, kind)
    _check(out, lse, q[0], k[0], v[0], kind)


@pytest.mark.parametrize("L", [1, 40])
@pytest.mark.parametrize("where", ["page", "tail"])
def test_scales_a_type_apart(where, L):
    """bf16: values of 2^-125 in one block (a scale of 2^-100, the smallest) or in the tail, beside some of 2^100: finite everywhere, and the sum of the weights is whole."""
    n = 650
    k, v = _rows(L, 1, 8, n, torch.bfloat16)
    v[:, :, 64:128] = v[:, :, 64:128].sign() * 2.0 ** 100
    near = slice(320, 384) if where == "page" else slice(640, 650)
    v[:, :, near] = v[:, :, near].sign() * 2.0 ** -125
    q = _queries(L, 1, 8, L, torch.bfloat16)
    out, lse = _attend(k, v, q, "int8")
    _check(out, lse, q[0], k[0], v[0], "int8")


def test_weights_are_rounded_once():
    """Where the second half of a block brings a query's sums to a new reference, the first half's weights, rounded already, lose nothing more.  All values are one number,
    of which a weighted mean is more only by the weights' rounding, 2^-11 of it at the most, and that does not take it to fp16's next number: it is held as 1.7457275390625, the
    middle above the number that this rounds to is more than 2^-11 of it away.  (One query of each wavefront has a score that calls for the new reference.)"""
    L, n = 256, 64 + 256
    g = torch.Generator().manual_seed(5)
    k = torch.zeros(1, 1, n, 128)
    k[..., 2] = -1                                            # (tokens that have no say)
    k[0, 0, :32], k[0, 0, 40] = 0, 0
    k[0, 0, 0, 0] = k[0, 0, 40, 1] = 1
    k[0, 0, 1:32, 3] = 1
    per = 128 ** 0.5 * 0.6931                                 # a unit of base 2
    q = torch.zeros(1, 1, L, 128)
    q[..., 2] = 40 * per
    top = 4 * torch.rand(L, generator=g)
    q[0, 0, :, 0], q[0, 0, :, 3], q[0, 0, :, 1] = top * per, (top - torch.rand(L, generator=g)) * per, (top + torch.rand(L, generator=g)) * per
    q[0, 0, 5::32, 1] += 12 * per
    v = torch.full((1, 1, n, 128), 1.751953125, dtype=torch.float16)
    held = float(plain.held(v[0], "int8")[0, 0, 0])
    up = float(plain.to_type(torch.tensor(held), torch.float16)) + 2.0 ** -11              # the middle above: fp16's numbers are 2^-10 apart
    assert held == 1.7457275390625 and up / held > 1 + 2.0 ** -11
    out = _filled(k.half(), v, [n], "int8").attend(0, q.half().to(DEV)).cpu().double()
    assert float(out.max()) < up, ((out > up).any(dim=-1).sum(), out.max())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("L", [1, 3, 17, 40, 130])
@pytest.mark.parametrize("at", [3, 40, 200, 400, 447, 500])
def test_a_token_that_outweighs_the_others_is_rounded_once(at, L, kind):
    """A token 2^-40 of whose weight all others have together: the outputs are what is held of its values, rounded to fp16 and nothing else but what 32 bits leave (the
    logarithm of a scale and its power: 2^-21, by which a value half-way between two fp16 numbers may go either way).  In either half of a block and in the tail."""
    n = 508
    k, v = _rows(at, 1, 2, n, torch.float16)
    k[..., 0] = 0
    k[0, :, at, 0] = 40
    q = _queries(L, 1, 8, L, torch.float16, size=0.7)
    q[..., 0] = 13.7
    out = _filled(k, v, [n], kind).attend(0, q.to(DEV))[0].cpu().double()
    want = plain.held(v[0], kind)[:, at].repeat_interleave(4, dim=0).expand(L, 8, 128)
    sees = torch.arange(n - L, n) >= at
    # half a step of fp16 at each value: 2^-11 of the power of two below it, 2^-25 for the smallest
    half = (2.0 ** (torch.frexp(want.abs()).exponent - 12).double()).clamp(min=2.0 ** -25)
    assert bool(sees.any()) and bool(((out - want).abs()[sees] <= (half + 2.0 ** -21 * want.abs())[sees]).all()), float(((out - want).abs() / half)[sees].max())


def _at_the_end(v, signs, by):
    """Values of bf16's largest magnitude and 0.97 of it, times `by`; their signs one for all, or another for each half of the tokens, each block of 64, each token."""
    t = torch.arange(v.shape[2])
    flip = {"all above": 0 * t, "all below": 0 * t + 1, "halves": (t >= v.shape[2] // 2).long(), "blocks": t // 64 % 2, "tokens": t % 2}[signs]
    size = torch.where(v > 0, 1.0, 0.97).to(v.dtype) * (torch.finfo(v.dtype).max * by)
    return torch.where(flip[None, None, :, None] > 0, -size, size)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("signs", ["all above", "all below", "halves", "blocks", "tokens"])
@pytest.mark.parametrize("by", [1.0, 2.0 ** -5])
def test_values_at_the_type_s_end(by, signs, kind):
    """bf16 values whose weighted sum passes 32 bits though their mean does not: a row in shares and by itself, among few queries and many, and rows with most of it in common."""
    dtype, n = torch.bfloat16, 3000
    k, v = _rows(51, 1, 2, n, dtype)
    v = _at_the_end(v, signs, by)
    for L in (1, 4, 40):
        q = _queries(52, 1, 8, L, dtype)
        out, lse = _filled(k, v, [n], kind).attend(0, q.to(DEV), return_lse=True)
        _check(out[0], lse[0], q[0], k[0], v[0], kind)
        out, lse = _attend(k, v, q, kind)
        _check(out, lse, q[0], k[0], v[0], kind)
    one = _filled(k, v, [n], kind)
    for rows in (3, 40):
        c = one.select([0] * rows)
        q = _queries(53, rows, 8, 2, dtype)
        out, lse = c.attend(0, q.to(DEV), return_lse=True, shared=True)
        for b in (0, rows - 1):
            _check(out[b], lse[b], q[b], k[0], v[0], kind)
        c.release()


@pytest.mark.parametrize("cap", [2.0 ** 40, 2.0 ** 100, 2.0 ** 125, 2.0 ** 127, 3.4e38])
@pytest.mark.parametrize("dtype", DTYPES)
def test_caps_that_cap_nothing(dtype, cap):
    """A cap past all scores by 2^30 changes them by 2^-60: the results are the definition's without one, up to the largest cap that 32 bits hold; few queries, many, and what rows have in common."""
    n = 700
    k, v = _rows(54, 1, 2, n, dtype)
    one = _filled(k, v, [n], "int8")
    c = one.select([0] * 3)
    for L, shared in ((1, False), (4, True), (40, False)):
        q = _queries(55, 3, 8, L, dtype)
        out, lse = c.attend(0, q.to(DEV), softcap=cap, shared=shared, return_lse=True)
        for b in range(3):
            _check(out[b], lse[b], q[b], k[0], v[0], "int8")


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_are_not_numbers(dtype):
    """They give what is not a number, from a row in shares, by itself and with most of it in common, among few queries and many; the others what the definition says."""
    n = 3000
    k, v = _rows(56, 1, 2, n, dtype)
    one = _filled(k, v, [n], "int8")
    c = one.select([0] * 3)
    for cache, rows, L, shared in ((one, 1, 1, False), (one, 1, 40, False), (c, 3, 1, False), (c, 3, 4, True), (c, 3, 40, False)):
        q = _queries(57, rows, 8, L, dtype)
        want = cache.attend(0, q.to(DEV), shared=shared, return_lse=True)
        bad = q.clone()
        bad[rows - 1, 5, L - 1] = float("nan")
        got = cache.attend(0, bad.to(DEV), shared=shared, return_lse=True)
        for x, y, at in zip(got, want, ((rows - 1, L - 1, 5), (rows - 1, 5, L - 1))):
            assert bool(torch.isnan(x[at]).all()), (rows, L, shared)
            x[at] = y[at]
        for b in range(rows):
            _check(got[0][b], got[1][b], q[b], k[0], v[0], "int8")
