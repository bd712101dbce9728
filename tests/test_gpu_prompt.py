"""GPU: attention of whole prompts in 16 bits against its definition in 64 bits (tests/prompt_rows.py)."""
import pytest
import torch

import prompt_rows as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def _inputs(seed, B, Hq, H, L, T, dtype):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, h, n, 128, generator=g) for h, n in ((Hq, L), (H, T), (H, T)))
    k[..., :4] *= 5
    v *= 0.2 + torch.rand(B, H, T, 1, generator=g)
    return (2 * q).to(dtype).to(DEV), k.to(dtype).to(DEV), v.to(dtype).to(DEV)


def _call(*args, **kw):
    from kvquant import prompt_attention
    return prompt_attention(*args, return_lse=True, **kw)


def _check(q, k, v, starts=None, cap=None, window=None, scaling=None, causal=True):
    given = dict(starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV))
    out, lse = _call(q, k, v, softcap=cap, window=window, scaling=scaling, causal=causal, **given)
    assert out.shape == (q.shape[0], q.shape[2], q.shape[1], 128) and out.dtype == q.dtype and lse.shape == q.shape[:3] and lse.dtype == torch.float32
    for b in range(q.shape[0]):
        plain.check(out[b], lse[b], *plain.attend(q[b], k[b], v[b], scaling=scaling, cap=cap, window=window, start=0 if starts is None else starts[b], causal=causal))
    return out, lse


SHAPES = [(1, 4, 1, 1, 1), (2, 8, 2, 63, 63), (1, 4, 4, 64, 64), (1, 7, 1, 65, 65), (1, 1, 1, 257, 257), (2, 6, 2, 200, 333), (1, 8, 1, 130, 40), (1, 4, 2, 1, 700),
          (1, 16, 2, 300, 300), (3, 28, 4, 127, 129), (1, 40, 2, 33, 100), (1, 32, 8, 1000, 1000), (1, 8, 8, 5, 3000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,H,L,T", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_shapes(B, Hq, H, L, T, dtype):
    _check(*_inputs(L + T, B, Hq, H, L, T, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("change", [dict(cap=30.0), dict(cap=100.0), dict(cap=0.7), dict(window=1), dict(window=64), dict(window=100, cap=20.0), dict(starts=[0, 17, 299]),
                                    dict(starts=[-5, 64, 1000], window=90), dict(causal=False), dict(causal=False, starts=[0, 100, 300], cap=5.0), dict(scaling=-0.05),
                                    dict(scaling=0.0), dict(scaling=0.5)], ids=str)
def test_what_is_seen_and_how(change, dtype):
    _check(*_inputs(3, 3, 6, 2, 300, 300, dtype), **change)
    _check(*_inputs(4, 3, 6, 2, 70, 300, dtype), **change)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed(dtype):
    """Sequences of their own lengths, empty ones and queries of none among them; keys of other lengths than the queries."""
    lengths = [0, 130, 1, 64, 0, 300, 63, 65, 2]
    begin, N = 3, sum([0, 130, 1, 64, 0, 300, 63, 65, 2]) + 3 + 9
    q, k, v = _inputs(5, 1, 6, 2, N, N, dtype)
    ends = torch.tensor([begin, *lengths]).cumsum(0)
    out, lse = _call(q, k, v, offsets=ends.to(torch.int32).to(DEV))
    for a, e in zip(ends.tolist(), ends.tolist()[1:]):
        plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, a:e], v[0, :, a:e]))
    for a, e in ((0, begin), (N - 9, N)):
        assert not out[0, a:e].any() and bool((lse[0, :, a:e] == -torch.inf).all())
    # chunks: more keys than queries, fewer, none; starts of their own
    keys = [5, 400, 300, 1, 64, 0, 1000, 63, 2]
    _, k, v = _inputs(6, 1, 6, 2, 1, sum(keys) + 7, dtype)
    key_ends = torch.tensor([4, *keys]).cumsum(0)
    starts = [0, 100, 0, 2, 0, 0, 990, 1, 0]
    for change in (dict(), dict(window=50, softcap=20.0), dict(causal=False)):
        out, lse = _call(q, k, v, offsets=ends.to(DEV), key_offsets=key_ends.to(DEV), starts=torch.tensor(starts, device=DEV), **change)
        want = dict(cap=change.get("softcap"), window=change.get("window"), causal=change.get("causal", True))
        for s, (a, e, x, y) in enumerate(zip(ends.tolist(), ends.tolist()[1:], key_ends.tolist(), key_ends.tolist()[1:])):
            plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, x:y], v[0, :, x:y], start=starts[s], **want))


def test_many_sequences():
    """More of them than lanes, most of one tile's queries or less."""
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 60, (200,), generator=g).tolist()
    ends = torch.tensor([0, *lengths]).cumsum(0)
    q, k, v = _inputs(9, 1, 4, 1, int(ends[-1]), int(ends[-1]), torch.bfloat16)
    out, lse = _call(q, k, v, offsets=ends.to(torch.int32).to(DEV))
    for a, e in zip(ends.tolist(), ends.tolist()[1:]):
        plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, a:e], v[0, :, a:e]))


@pytest.mark.parametrize("scaling", [None, -0.02], ids=["plain", "negative"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_more_tiles_than_workgroups_take_at_once(dtype, scaling):
    """Sequences of many lengths, empty ones among them, chunks that see nothing, infinite values behind what is seen; the same bits twice."""
    lengths = [700, 0, 333, 1, 0, 900, 64, 63, 257, 500, 128, 2, 31, 640, 0, 411]
    keys = [700, 5, 333, 1, 0, 950, 64, 0, 100, 900, 128, 2, 31, 640, 64, 411]
    ends, key_ends = torch.tensor([7, *lengths]).cumsum(0), torch.tensor([3, *keys]).cumsum(0)
    N, M = int(ends[-1]) + 11, int(key_ends[-1]) + 2
    q, k, v = _inputs(12, 1, 32, 8, N, M, dtype)
    v[0, :, 3 + 650] = float("inf")                                     # of the first sequence, whose first queries do not see it
    call = dict(offsets=ends.to(torch.int32).to(DEV), key_offsets=key_ends.to(torch.int32).to(DEV), scaling=scaling)
    out, lse = _call(q, k, v, **call)
    for a, e, x, y in zip(ends.tolist(), ends.tolist()[1:], key_ends.tolist(), key_ends.tolist()[1:]):
        plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, x:y], v[0, :, x:y], scaling=scaling))
    for a, e in ((0, 7), (N - 11, N)):
        assert not out[0, a:e].any() and bool((lse[0, :, a:e] == -torch.inf).all())
    for _ in range(3):
        again, lse_again = _call(q, k, v, **call)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16)) and torch.equal(lse.view(torch.int32), lse_again.view(torch.int32))


@pytest.mark.parametrize("change", [dict(), dict(starts=[4321]), dict(window=5000), dict(causal=False)], ids=str)
def test_tiles_that_leave_units_without_one(change):
    """Long chunks whose keys are shared out, two unequal shares among them."""
    _check(*_inputs(16, 1, 24, 24, 2000, 9000, torch.float16), **change)
    _check(*_inputs(17, 1, 32, 8, 1600, 6500, torch.bfloat16), **change)


@pytest.mark.parametrize("change", [dict(window=1000), dict(window=130, cap=20.0), dict(window=3000, starts=[7500])], ids=str)
def test_few_queries_over_a_window(change):
    """A window's blocks shared out, fewer of them than the keys have."""
    _check(*_inputs(18, 1, 32, 8, 100, 8000, torch.float16), **change)
    _check(*_inputs(19, 1, 14, 2, 1, 8000, torch.bfloat16), **change)


def test_more_tiles_in_rows():
    _check(*_inputs(13, 2, 32, 8, 1500, 1500, torch.bfloat16), starts=[0, 333])
    _check(*_inputs(14, 17, 24, 8, 260, 400, torch.float16), window=90)
    q, k, v = _inputs(15, 1, 32, 8, 4200, 1, torch.float16)             # most see nothing
    _check(q, k, v)


@pytest.mark.parametrize("bad", [[0, 50, 40, 100], [-7, 30, 60, 100], [0, 30, 60, 500], [90, 50, 20, 0], [0, 2 ** 31 - 1, -2 ** 31, 100], [100, 100, 100, 100]], ids=str)
def test_offsets_that_do_not_ascend_stay_within_the_tensors(bad):
    q, k, v = _inputs(10, 1, 4, 2, 100, 100, torch.float16)
    guard = torch.full((3, 100, 4, 128), 7.0, dtype=torch.float16, device=DEV)
    from kvquant import _lib
    import ctypes as C
    offsets = torch.tensor(bad, dtype=torch.int32, device=DEV)
    a = _lib.PromptAttend(*(x for t in (q, k, v) for x in (t.data_ptr(), *t.stride()[:3])), guard[1].data_ptr(), 0, offsets.data_ptr(), 0, 0, 0, 0, 0, 3, 100, 100, 4, 2, 1, 0, 0.1, 0.0)
    _lib.check(_lib.lib.odmkv_prompt_attend(C.byref(a), _lib.stream_ptr(q.device)))
    assert bool((guard[0] == 7).all()) and bool((guard[2] == 7).all()) and bool(torch.isfinite(guard).all())


SOUND = [0, 30, 70, 100]


@pytest.mark.parametrize("bad", [[0, 100, -2 ** 31, 120], [0, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [150, -2 ** 31, 5, 60], [-2 ** 31, -2 ** 31, 200, 2 ** 31 - 1], [200, 0, 300, -1],
                                 [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [0, 50, 40, 150]], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_key_offsets_that_do_not_ascend_beside_sound_ones(bad, dtype):
    """Sound queries: each sequence sees what its two offsets say of the keys there are, and nothing of what lies in front of and behind them."""
    q, inner_k, inner_v = _inputs(31, 1, 6, 2, 100, 150, dtype)
    room = 70000                                                        # NaN on both sides: whoever reads them shows it
    k, v = (torch.full((1, 2, room + 150 + room, 128), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    for to, x in ((k, inner_k), (v, inner_v)):
        to[:, :, room:room + 150] = x
    k, v = k[:, :, room:room + 150], v[:, :, room:room + 150]
    offsets, key_offsets = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (SOUND, bad))
    for how in (dict(), dict(causal=False), dict(window=20, cap=30.0)):
        out, lse = _call(q, k, v, offsets=offsets, key_offsets=key_offsets, causal=how.get("causal", True), window=how.get("window"), softcap=how.get("cap"))
        for s in range(3):
            a, e = SOUND[s:s + 2]
            x = min(max(bad[s], 0), 150)
            y = max(min(max(bad[s + 1], 0), 150), x)
            plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, x:y], v[0, :, x:y], **how))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_where_nobody_looks(dtype):
    """In padding, in other sequences, behind a query's end and in front of its window: a query's result is what it is without them; whoever sees them gets them."""
    q, k, v = _inputs(11, 2, 6, 2, 150, 150, dtype)
    starts = torch.tensor([40, 0], dtype=torch.int32, device=DEV)
    clean = _call(q, k, v, starts=starts)
    for x, t in ((k, 3), (v, 39), (v, 0)):
        x[0, :, t] = float("nan") if t else float("inf")
    dirty = _call(q, k, v, starts=starts)
    for b in range(2):
        want = plain.attend(q[b], k[b].nan_to_num(0, 0, 0), v[b].nan_to_num(0, 0, 0), start=[40, 0][b])
        plain.check(clean[0][b], clean[1][b], *want)
        plain.check(dirty[0][b], dirty[1][b], *want)
    # (bits may differ: what is spoilt is summed again with weights in 32 bits.  Both are as far from the definition as they may be, so twice that from one another: checked above)
    assert torch.equal(clean[1], dirty[1])
    # packed: neighbours of the poisoned one
    ends = torch.tensor([0, 70, 75, 150], dtype=torch.int32, device=DEV)
    q, k, v = _inputs(12, 1, 6, 2, 150, 150, dtype)
    v[0, :, 70:75], k[0, :, 72] = float("nan"), float("inf")
    out, lse = _call(q, k, v, offsets=ends)
    for a, e in ((0, 70), (75, 150)):
        plain.check(out[0, a:e], lse[0, :, a:e], *plain.attend(q[0, :, a:e], k[0, :, a:e], v[0, :, a:e]))
    assert bool(torch.isnan(out[0, 70:75]).all())
    # a later token's, and one that a window has passed by
    q, k, v = _inputs(13, 1, 6, 2, 150, 150, dtype)
    v[0, 0, 100, 5], v[0, 1, 100, 77], v[0, 1, 20, 3] = float("nan"), float("-inf"), float("inf")
    out, lse = _check(q, k, v, window=30)
    assert bool(torch.isfinite(out[0, :100, :3]).all()) and bool(torch.isnan(out[0, 100:130, :3, 5]).all()) and bool(torch.isfinite(out[0, 130:, :3]).all())
    _check(q, k, v)
    # a key that is not a number: whoever sees it
    k[0, 0, 50, 0] = float("nan")
    out, _ = _call(q, k, v)
    assert bool(torch.isfinite(out[0, :50, :3]).all()) and bool(torch.isnan(out[0, 50:, :3]).all())


def test_values_at_the_type_s_end():
    """bf16 values whose sum passes 32 bits though their mean does not; fp16 ones."""
    for dtype in DTYPES:
        q, k, v = _inputs(14, 1, 4, 2, 200, 200, dtype)
        v = torch.where(v > 0, 1.0, 0.98).to(dtype) * torch.finfo(dtype).max
        _check(q, k, v)
        _check(q, k, -v)


SIGNS = ("all above", "all below", "halves", "blocks", "tokens")


def _at_the_end(v, signs, by=1.0):
    """Values of the type's largest magnitude and 0.98 of it, times `by`; their signs one for all, or another for each half of the tokens, each block of 64, each token."""
    t = torch.arange(v.shape[2], device=v.device)
    flip = {"all above": 0 * t, "all below": 0 * t + 1, "halves": (t >= v.shape[2] // 2).long(), "blocks": t // 64 % 2, "tokens": t % 2}[signs]
    size = torch.where(v > 0, 1.0, 0.98).to(v.dtype) * (torch.finfo(v.dtype).max * by)
    return torch.where(flip[None, None, :, None] > 0, -size, size)


@pytest.mark.parametrize("signs", SIGNS)
@pytest.mark.parametrize("shape", [(1, 8, 1, 1, 20000), (1, 4, 2, 3, 6000), (2, 6, 2, 5, 3000), (1, 24, 24, 2000, 9000)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_type_s_end_in_shares(dtype, shape, signs):
    """Few queries over many keys: a tile's keys are shared out, and the shares' results, of values that 32 bits just hold, are put together."""
    from kvquant import _lib
    B, Hq, H, L, T = shape
    assert _lib.lib.odmkv_prompt_attend_workspace_bytes(0, B, Hq, H, L, T, 1, 0, 0.0) >= 2 * B * L * Hq * 129 * 4
    q, k, v = _inputs(32, *shape, dtype)
    _check(q, k, _at_the_end(v, signs))
    if dtype == torch.bfloat16 and L < 10:
        _check(q, k, _at_the_end(v, signs, by=2.0 ** -6))               # (what 64 shares of one sign add up to)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("shape", [(1, 4, 2, 32, 32), (1, 2, 1, 1, 1000), (1, 8, 1, 3, 9000), (2, 4, 4, 200, 200), (1, 32, 8, 700, 700)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_mean_of_the_type_s_largest_is_that(dtype, shape, sign):
    """All values are the type's largest (or its negative), and weights round upwards: their sum over the sum of what they were passes one, the result does not pass the type's end.
    One key in 64 outweighs the others by nearly two: of a weight of 2^8 they have 128.069, in fp16 128.125, and of a weight of 1 just above a half and a step's half, in bf16 a half and a step."""
    B, Hq, H, L, T = shape
    q, k, v = (torch.zeros(B, h, n, 128, dtype=dtype, device=DEV) for h, n in ((Hq, L), (H, T), (H, T)))
    q[..., 0], k[:, :, ::64, 0] = 1, 1
    v[:] = sign * torch.finfo(dtype).max
    out, _ = _check(q, k, v, scaling=0.69314718 * (0.99922 if dtype == torch.float16 else 0.99434))
    none = max(0, L - T)
    assert bool((out[:, none:] == sign * torch.finfo(dtype).max).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_beside_the_type_s_largest(dtype):
    """Whoever sees an infinite value, or both infinities, or a NaN, gets what the definition says, in one share and in several; the others stay within the type's end."""
    for shape in ((1, 4, 2, 150, 150), (1, 4, 2, 40, 7000)):
        q, k, v = _inputs(33, *shape, dtype)
        v = _at_the_end(v, "tokens")
        last = shape[4]
        v[0, 0, last - 30, 3], v[0, 0, last - 20, 3], v[0, 1, last - 25, 7], v[0, 1, 5, 9] = float("inf"), float("-inf"), float("nan"), float("-inf")
        _check(q, k, v)
        _check(q, k, v, window=12)


@pytest.mark.parametrize("shape", [(1, 4, 2, 150, 150), (1, 4, 2, 3, 7000)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_are_not_numbers(dtype, shape):
    """They give what is not a number, in one share and in several, and their neighbours what they gave without them."""
    q, k, v = _inputs(34, *shape, dtype)
    for bad in (float("nan"), float("inf")):
        q[0, 1, 2, 5], k[..., 5] = bad, 0                               # (infinite times 0 is not a number)
        out, lse = _call(q, k, v)
        assert bool(torch.isnan(out[0, 2, 1]).all()) and bool(torch.isnan(lse[0, 1, 2]))
        clean = q.clone()
        clean[0, 1, 2, 5] = 0
        want, want_lse, tol, lse_tol = plain.attend(clean[0], k[0], v[0])
        out[0, 2, 1], lse[0, 1, 2] = want[2, 1].to(dtype), want_lse[1, 2].float()
        plain.check(out[0], lse[0], want, want_lse, tol, lse_tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_rise(dtype):
    """Every later key outscores the ones before by far, or falls behind: the reference moves many times, or never."""
    q, k, v = _inputs(15, 1, 4, 2, 500, 500, dtype)
    for ramp in (torch.linspace(0, 40, 500), torch.linspace(40, 0, 500), torch.linspace(-300, 300, 500)):
        q[..., 0], k[..., 0] = 10.0, ramp.to(dtype).to(DEV)
        _check(q, k, v)
        _check(q, k, v, cap=50.0)


@pytest.mark.parametrize("cap", [2.0 ** 40, 2.0 ** 100, 2.0 ** 125, 2.0 ** 127, 3.4e38])
@pytest.mark.parametrize("dtype", DTYPES)
def test_caps_that_cap_nothing(dtype, cap):
    """A cap past all scores by 2^30 changes them by 2^-60: the results are the definition's without one, up to the largest cap that 32 bits hold."""
    for shape in ((1, 6, 2, 150, 150), (1, 8, 1, 2, 5000)):
        q, k, v = _inputs(20, *shape, dtype)
        out, lse = _call(q, k, v, softcap=cap)
        plain.check(out[0], lse[0], *plain.attend(q[0], k[0], v[0]))


def test_strides_types_and_bits():
    """Slices of one projection, rows that do not start on 16 bytes, one row for all heads: the same bits as of copies; a call made twice gives the same bits."""
    g = torch.Generator().manual_seed(16)
    wide = torch.randn(2, 130, (8 + 2 * 2) * 128, generator=g).to(torch.bfloat16).to(DEV)
    q, k, v = (x.view(2, 130, -1, 128).transpose(1, 2) for x in wide.split([8 * 128, 2 * 128, 2 * 128], dim=2))
    want = _call(q.contiguous(), k.contiguous(), v.contiguous())
    for got in (_call(q, k, v), _call(q, k, v)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(2, 8, 130, 129, dtype=torch.bfloat16, device=DEV)[..., 1:]
    odd.copy_(q)
    assert torch.equal(_call(odd, k, v)[0], want[0])
    one = k[:, :1].expand(2, 2, 130, 128)
    assert torch.equal(_call(q, one, v)[0], _call(q, one.contiguous(), v)[0])


def test_no_queries_and_no_keys():
    q, k, v = _inputs(17, 2, 4, 2, 5, 0, torch.float16)
    out, lse = _call(q, k, v)
    assert out.shape == (2, 5, 4, 128) and not out.any() and bool((lse == -torch.inf).all())
    out, lse = _call(q[:, :, :0], k, v)
    assert out.shape == (2, 0, 4, 128) and lse.shape == (2, 4, 0)


def test_a_long_prompt():
    """4999 tokens of 28 heads over 4: rows here and there, in 64 bits."""
    q, k, v = _inputs(18, 1, 28, 4, 4999, 4999, torch.bfloat16)
    out, lse = _call(q, k, v)
    for i in (0, 63, 64, 1234, 4096, 4998):
        plain.check(out[0, i:i + 1], lse[0, :, i:i + 1], *plain.attend(q[0, :, i:i + 1], k[0, :, :i + 1], v[0, :, :i + 1]))


def test_captured_and_on_another_stream():
    """A captured call with shares of its own scratch: every replay is the eager call, on inputs that change in between."""
    for shape in ((1, 8, 2, 200, 200), (1, 4, 1, 3, 2000)):
        q, k, v = _inputs(19, *shape, torch.float16)
        qs, ks, vs = q.clone(), k.clone(), v.clone()
        _call(qs, ks, vs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _call(qs, ks, vs)
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other):
            second = _call(ks[:, :1].expand(-1, shape[1], -1, -1)[:, :, :shape[3]], ks, vs)
        for i in range(3):
            x = _inputs(20 + i, *shape, torch.float16)
            for to, y in zip((qs, ks, vs), x):
                to.copy_(y)
            graph.replay()
            other.replay()
            graph.replay()
            want, want2 = _call(*x), _call(x[1][:, :1].expand(-1, shape[1], -1, -1)[:, :, :shape[3]], *x[1:])
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(second[0], want2[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = _call(qs, ks, vs)
        side.synchronize()
        assert torch.equal(there[0], got[0])


def test_what_would_be_recorded_is_refused():
    """Gradients while they are recorded, tangents with and without: of each operand by itself, by the native call and by the other."""
    from torch.autograd import forward_ad
    from kvquant import prompt_attention
    given = _inputs(41, 1, 4, 2, 10, 10, torch.float16)
    odd = torch.zeros(1, 4, 10, 129, dtype=torch.float16, device=DEV)[..., 1:]              # (not by the native call)
    want = prompt_attention(*given)
    for first in (given[0], odd):
        for i in range(3):
            args = [first, *given[1:]]
            args[i] = args[i].detach().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradients"):
                prompt_attention(*args)
            with forward_ad.dual_level(), torch.no_grad():
                args[i] = forward_ad.make_dual(args[i].detach(), torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="no tangents"):
                    prompt_attention(*args)
    with forward_ad.dual_level():                                                            # (plain tensors among dual numbers)
        assert torch.equal(prompt_attention(*given), want)


def test_refusals():
    from kvquant import prompt_attention
    q, k, v = _inputs(21, 2, 4, 2, 10, 10, torch.float16)
    i32 = dict(dtype=torch.int32, device=DEV)
    two = torch.tensor([0, 5, 10], **i32)
    for args, kw, says in (((q[0], k, v), {}, "queries must be"), ((q, k[..., :64], v), {}, "keys must be"), ((q.float(), k, v), {}, "float16 or bfloat16"),
                           ((q, k.bfloat16(), v), {}, "one type"), ((q, k, v[:, :, :5]), {}, "values"), ((q, k[:1], v[:1]), {}, "rows"), ((q[:, :3], k, v), {}, "3 query heads"),
                           ((q, k, v), dict(softcap=0.0), "softcap"), ((q, k, v), dict(softcap=float("nan")), "softcap"), ((q, k, v), dict(window=0), "window"),
                           ((q, k, v), dict(window=5, causal=False), "window"), ((q, k, v), dict(offsets=two), "packed"), ((q[:1], k[:1], v[:1]), dict(key_offsets=two), "offsets"),
                           ((q[:1], k[:1], v[:1]), dict(offsets=two[:1]), "offsets"), ((q[:1], k[:1], v[:1]), dict(offsets=two.float()), "whole numbers"),
                           ((q[:1], k[:1], v[:1]), dict(offsets=two.cpu()), "lie on"), ((q[:1], k[:1], v[:1]), dict(offsets=[0, 10]), "offsets"),
                           ((q[:1, :, :4], k[:1], v[:1]), dict(offsets=two), "key_offsets"), ((q, k, v), dict(starts=torch.zeros(3, **i32)), "starts")):
        with pytest.raises(ValueError, match=says):
            prompt_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        prompt_attention(q.cpu(), k, v)
    with pytest.raises(RuntimeError, match="no gradients"):
        prompt_attention(q, k.clone().requires_grad_(), v)
    with torch.no_grad():
        prompt_attention(q, k.clone().requires_grad_(), v)
