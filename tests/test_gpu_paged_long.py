"""GPU: attention over the paged 8-bit cache where one wavefront goes through more than 64 blocks of a row, whose pages and scales it looks up 64 at a time."""
import pytest
import torch

import paged_rows as plain
from test_gpu_paged_cache import DEV, _cache, _queries, _rows

pytestmark = pytest.mark.gpu


def _long_row(seed, H, n, dtype):
    """A row whose later blocks' values are larger than the first ones', some of them by far, and smaller again."""
    k, v = _rows(seed, 1, H, n, dtype)
    at = torch.arange(n).view(1, 1, n, 1) / n
    by = torch.where(at < 0.4, 2.0 ** -5, torch.where(at < 0.8, torch.ones(()), torch.tensor(2.0 ** -3)))
    by = torch.where((at > 0.85) & (at < 0.86), torch.tensor(2.0 ** 4), by)
    return k, (v.float() * by).to(dtype)


def _row_against_the_rest(B, H, Hq, n, L, kind, dtype, few=40):
    """A batch whose first row is long and the others short, so that a workgroup has a whole row to itself: the first row against the definition."""
    k, v = _long_row(n, H, n, dtype)
    c = _cache(B, H, n + 10, pages=n // 64 + B * (few // 64 + 1), kind=kind, dtype=dtype)
    kd, vd = (x.to(DEV).expand(B, H, n, 128) for x in (k, v))
    c.append(kd, vd, [n] + [few] * (B - 1))
    q = _queries(L, B, Hq, L, dtype, size=1.0)
    out, lse = c.attend(0, q.to(DEV), return_lse=True)
    for b, m in ((0, n), (B - 1, few)):
        want, wl, tol, tl = plain.attend(q[b], plain.held(k[0, :, :m], kind), plain.held(v[0, :, :m], kind))
        got, gl = out[b].cpu().double(), lse[b].cpu().double()
        ok = torch.isfinite(wl)
        assert torch.isfinite(got).all() and torch.equal(torch.isfinite(gl), ok) and ((gl - wl).abs()[ok] <= tl[ok] + 2.0 ** -23 * wl.abs()[ok]).all()
        assert ((got - want).abs() <= tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)).all(), (b, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("kind,dtype", [("int8", torch.float16), ("e4m3", torch.bfloat16)])
@pytest.mark.parametrize("L", [1, 3])
def test_a_step_over_a_row_of_300_blocks_in_one_workgroup(L, kind, dtype):
    """64 rows of 8 heads: a workgroup of four wavefronts takes a row, 78 blocks and more a wavefront."""
    _row_against_the_rest(64, 8, 8, 20011, L, kind, dtype)


@pytest.mark.parametrize("kind,dtype", [("int8", torch.bfloat16), ("e4m3", torch.float16)])
@pytest.mark.parametrize("L", [17, 40, 130])
def test_many_queries_over_a_row_of_80_blocks_in_one_workgroup(L, kind, dtype):
    """65 rows of 4 heads: no row's blocks are shared out, a workgroup goes through all of them."""
    _row_against_the_rest(65, 4, 4, 5333, L, kind, dtype, few=200)


def test_a_step_over_a_row_of_2000_blocks():
    """Eight wavefronts a workgroup: one row of 2 heads and 131071 tokens, windowed and not."""
    n, H = 131071, 2
    k, v = _long_row(5, H, n, torch.float16)
    c = _cache(1, H, n + 5)
    c.append(k.to(DEV), v.to(DEV))
    q = _queries(1, 1, 2 * H, 1, torch.float16, size=1.0)
    for how in ({}, dict(window=70000), dict(starts=torch.tensor([100000], dtype=torch.int32))):
        out, lse = c.attend(0, q.to(DEV), return_lse=True, **{name: x.to(DEV) if torch.is_tensor(x) else x for name, x in how.items()})
        args = dict(how, starts=how["starts"][0]) if "starts" in how else how
        want, wl, tol, tl = plain.attend(q[0], plain.held(k[0], "int8"), plain.held(v[0], "int8"), **args)
        got = out[0].cpu().double()
        assert ((lse[0].cpu().double() - wl).abs() <= tl + 2.0 ** -23 * wl.abs()).all()
        assert ((got - want).abs() <= tol + 2.0 ** -11 * (want.abs() + tol)).all()
