"""The row operators by where their rows lie: rows that fill their threads exactly, and x, residual, h and q that
stand apart from one another in their chunks of 8 elements (what a packed odd width beside codes on 16-byte
rows gives).  Tolerances as in test_gpu_operators.py."""
from __future__ import annotations

import pytest

from glypr_b200 import api
from .test_gpu_operators import DT, EPS, FLOOR, TINY, U, buffer, check_codes, filled, norm_want, ptr, rows_of, run_quantize

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    api.load_library()
    yield


def run_norm(x, res, post, gain, h, q, s, xd, hd, qd):
    m, n = x.shape
    api.norm_residual_q8(m, n, ptr(x), DT[xd], ptr(q), DT[qd], ptr(s), gain=ptr(gain), post_gain=ptr(post),
                         residual=ptr(res), h=ptr(h), h_dtype=DT[hd], eps=EPS, ld_x=x.stride(0),
                         ld_residual=res.stride(0) if res is not None else 0, ld_h=h.stride(0), ld_q=q.stride(0))


def gains(h, seed):
    return rows_of(1, h, seed, 0.0)[0] * 0.2 + 1


@pytest.mark.parametrize("h", [64, 128, 256, 512, 768, 1024, 1280, 2048, 4096, 5120, 6144, 8192, 12288, 16384])
@pytest.mark.parametrize("xd,hd,qd", [("f16", "bf16", "i8"), ("f32", "f32", "e4m3"), ("bf16", "f16", "e4m3")])
def test_rows_that_fill_their_threads(h, xd, hd, qd):
    for m, post_on in ((1, True), (37, True), (130, False)):
        x, res = filled(rows_of(m, h, h + m, 0.5), xd), filled(2 * rows_of(m, h, h + m + 1, 0.5), hd)
        post, gain = gains(h, 1) if post_on else None, gains(h, 2)
        hout, q, s = buffer(m, h, hd), buffer(m, h, qd), torch.empty(m, device="cuda")
        run_norm(x, res, post, gain, hout, q, s, xd, hd, qd)
        h_want, n_want, mag, n_mag = norm_want(x, res, post, gain, 1.0)
        err = (hout.double() - h_want).abs()
        assert (err <= U[hd] * h_want.abs() + 2.0 ** -18 * mag + TINY[hd]).all()
        check_codes(q, s, n_want, qd, n_mag)
        run_quantize(x, q, s, xd, qd)
        check_codes(q, s, x, qd)


# (pad, offset) of x, residual, h and q: one of them apart, then several
APART = {
    "q": ((0, 0), (0, 0), (0, 0), None),
    "q by a row": ((0, 0), (0, 0), (0, 0), (3, 0)),
    "h": ((0, 0), (0, 0), (0, 1), (0, 0)),
    "residual": ((0, 0), (1, 0), (0, 0), (0, 0)),
    "x": ((5, 3), (0, 0), (0, 0), (0, 0)),
    "all": ((1, 2), (2, 1), (3, 5), (4, 7)),
}


@pytest.mark.parametrize("where", APART)
@pytest.mark.parametrize("h", [5, 64, 203, 256, 771, 2048, 2051, 8001, 8192, 20003, 32768])
@pytest.mark.parametrize("xd,hd,qd", [("f16", "bf16", "i8"), ("bf16", "bf16", "e4m3"), ("f32", "f16", "i8")])
def test_operands_apart_in_their_chunks(h, xd, hd, qd, where):
    """Rows of zeros, of a NaN and of an infinity among them; nothing is written beside the rows."""
    m = 21
    px, pr, ph, pq = APART[where]
    if pq is None:  # codes on 16-byte rows, as the product wants them; apart for a width that is not
        pq = ((-h) % 16, 0) if h % 16 else (0, 1)
    x64, r64 = rows_of(m, h, h, 0.5), 2 * rows_of(m, h, h + 1, 0.5)
    x64[3], r64[3] = 0, 0
    x64[7, h - 1] = float("nan")
    r64[11, h // 2] = float("inf")
    x64[11, h // 2] = float("-inf")
    clean = [i for i in range(m) if i not in (7, 11)]
    x, res = filled(x64, xd, *px), filled(r64, hd, *pr)
    for post_on, res_on in ((True, True), (False, True), (True, False)):
        post, gain = gains(h, 1) if post_on else None, gains(h, 2)
        hout, q, s = buffer(m, h, hd, *ph, fill=7), buffer(m, h, qd, *pq, fill=0x21), torch.empty(m, device="cuda")
        whole = torch.as_strided(q.view(torch.uint8), (m, q.stride(0)), (q.stride(0), 1))
        run_norm(x, res if res_on else None, post, gain, hout, q, s, xd, hd, qd)
        h_want, n_want, mag, n_mag = norm_want(x[clean], res[clean] if res_on else None, post, gain, 1.0)
        err = (hout[clean].double() - h_want).abs()
        assert (err <= U[hd] * h_want.abs() + 2.0 ** -18 * mag + TINY[hd]).all()
        check_codes(q[clean], s[clean], n_want, qd, n_mag)
        assert (q[3].float() == 0).all() and s[3] == FLOOR
        assert torch.isnan(q.float() * s[:, None])[[7, 11]].all()
        assert (whole[:, h:] == 0x21).all()
    q, s = buffer(m, h, qd, *pq, fill=0x21), torch.empty(m, device="cuda")
    whole = torch.as_strided(q.view(torch.uint8), (m, q.stride(0)), (q.stride(0), 1))
    run_quantize(x, q, s, xd, qd)
    check_codes(q[clean], s[clean], x[clean], qd)
    assert (q[3].float() == 0).all() and s[3] == FLOOR
    assert torch.isnan(q.float() * s[:, None])[[7, 11]].all()
    assert (whole[:, h:] == 0x21).all()


@pytest.mark.parametrize("h", [771, 1152, 2051])
def test_in_place_with_codes_apart(h):
    m = 37
    x, res = filled(rows_of(m, h, 1), "f16"), filled(rows_of(m, h, 2), "bf16")
    outs = []
    for inplace in (False, True):
        r = res.clone()
        hout = r if inplace else torch.empty_like(r)
        q, s = buffer(m, h, "i8", 3, 1), torch.empty(m, device="cuda")
        run_norm(x, r, None, gains(h, 3), hout, q, s, "f16", "bf16", "i8")
        outs.append((q.clone(), s, hout))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
