"""The row operators at the ends of f32's range: rows of zeros without an eps, rows whose squares f32 cannot hold,
rows smaller than a quotient by them."""
from __future__ import annotations

import pytest

from glypr_b200 import api

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = api.DTYPES
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -100
# widths of every form: 8 lanes to 1,024 threads per row, whole lanes, off chunk boundaries
WIDTHS = [8, 64, 77, 256, 512, 768, 771, 1152, 1543, 2048, 5000, 12000, 20001]


@pytest.fixture(scope="module", autouse=True)
def _lib():
    api.load_library()
    yield


def ptr(t):
    return 0 if t is None else t.data_ptr()


def randn(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def norm(x, qd, eps, post=None, res=None, gain=None, apart=False):
    """(codes as f32, scale, h); apart: q off x's place in its chunks of 8, which takes the kernel for any
    alignment."""
    m, h = x.shape
    hout = torch.full_like(x, float("nan"))
    flat = torch.zeros(m * h + 16, dtype=torch.int8, device="cuda")
    q = flat[1 if apart else 0:][:m * h].view(m, h).view(TORCH[qd])
    s = torch.empty(m, device="cuda")
    xd = next(k for k, t in TORCH.items() if t == x.dtype)
    api.norm_residual_q8(m, h, ptr(x), DT[xd], ptr(q), DT[qd], ptr(s), gain=ptr(gain), post_gain=ptr(post),
                         residual=ptr(res), h=ptr(hout), h_dtype=DT[xd], eps=eps)
    return q.float(), s, hout


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("qd", ["i8", "e4m3"])
@pytest.mark.parametrize("h", WIDTHS)
def test_zero_rows_without_an_eps(h, qd, apart):
    """Codes 0 and the smallest scale, as for any other eps; the rows beside them are as ever."""
    x = randn(h, 6, h).bfloat16()
    x[1] = 0
    x[4] = 0
    post = randn(h + 1, h).abs() + 0.5
    for p in (None, post):
        q, s, hout = norm(x, qd, 0.0, post=p, apart=apart)
        q1, s1, h1 = norm(x, qd, 1e-30, post=p, apart=apart)
        assert (q[[1, 4]] == 0).all() and (s[[1, 4]] == FLOOR).all() and (hout[[1, 4]] == 0).all()
        assert torch.equal(q, q1) and torch.equal(s, s1) and torch.equal(hout, h1)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("h", WIDTHS)
def test_small_rows_without_an_eps(h, apart):
    """Rows of 1e-15 (squares of 1e-30) have the norm of the same rows times 2^50."""
    x = randn(h, 5, h) * 1e-15
    q, s, _ = norm(x, "i8", 0.0, apart=apart)
    q1, s1, _ = norm(x * 2.0 ** 50, "i8", 0.0, apart=apart)
    # the squares' sum and eps = 2^-126 against 1e-30: the statistic to 2^-22, codes apart by one step at most
    assert ((s / s1 - 1).abs() <= 2.0 ** -20).all()
    assert ((q - q1).abs() <= 1).all() and (q != q1).float().mean() < 1e-3


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype,qd", [("f32", "i8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("h", WIDTHS)
def test_rows_whose_squares_overflow(h, dtype, qd, apart):
    """Finite rows of 2^70: no zeros in place of their norm, but a scale of NaN; the rows beside them as ever."""
    x = randn(h, 6, h)
    x[2] *= 2.0 ** 70
    x[5, h // 2] = 2.0 ** 100
    x = x.to(TORCH[dtype])
    clean, big = [0, 1, 3, 4], [2, 5]
    post, res = randn(h + 1, h).abs() + 0.5, randn(h + 2, 6, h).to(TORCH[dtype])
    for p in (None, post):
        q, s, hout = norm(x, qd, 1e-6, post=p, res=res, apart=apart)
        assert torch.isnan(s[big]).all() and torch.isfinite(s[clean]).all()
        assert torch.isnan(q[big] * s[big, None]).all()
        assert torch.isfinite(hout[clean]).all()
        if p is None:
            assert torch.equal(hout, (x.float() + res.float()).to(x.dtype))
        q1, s1, h1 = norm(x[clean].contiguous(), qd, 1e-6, post=p, res=res[clean].contiguous(), apart=apart)
        if h % 8 == 0 or apart:  # (else the rows' places, and so the order of their sums, differ)
            assert torch.equal(q[clean], q1) and torch.equal(s[clean], s1)
    # up to there the norm is the norm
    y = randn(h, 3, h) * 2.0 ** 55
    q, s, _ = norm(y, "i8", 1e-6, apart=apart)
    q1, s1, _ = norm(y * 2.0 ** -55, "i8", 0.0, apart=apart)
    assert torch.equal(q, q1) and ((s / s1 - 1).abs() <= 2.0 ** -22).all()


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("qd", ["i8", "e4m3"])
@pytest.mark.parametrize("h", WIDTHS)
def test_rows_below_the_factor_of_their_codes(h, qd, apart):
    """Codes and scales stand for the row's norm, or the scale is NaN: no other values.  Gains of 2^-75 let a
    row of ordinary size come that near to zero, an eps of 0 one that is small itself."""
    x = randn(h, 8, h) * 2.0 ** torch.tensor([-40.0, -44, -48, -52, -55, -58, -60, -62], device="cuda")[:, None]
    gain = torch.full((h,), 2.0 ** -72, device="cuda")
    q, s, _ = norm(x, qd, 0.0, gain=gain, apart=apart)
    # the norm of x in 64 bits, its gain left out: 2^-72 of it is far above the smallest scale
    n = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 2.0 ** -126)
    v = q.double() * s.double()[:, None] * 2.0 ** 72
    top = n.abs().amax(1, keepdim=True)
    step = 1 / 127 if qd == "i8" else 1 / 14  # e4m3: 2^-3 of a binade, of 448 at most 32
    fine = torch.isnan(s)[:, None] | ((v - n).abs() <= 0.51 * step * top)
    assert fine.all()
    assert torch.isfinite(s[:2]).all()  # |h gain| of 2^-112 and 2^-116 have their codes


@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("m", [4, 40, 200])
@pytest.mark.parametrize("gated", [False, True])
def test_scales_whose_product_leaves_the_range(m, gated, off):
    """x_scale * w_scale of 1e-42 and of 1e42, with sums that bring the value back: operands on and off 16-byte
    rows."""
    n, k = 72, 96
    g = torch.Generator(device="cuda")
    g.manual_seed(m)

    def codes(rows):
        flat = torch.zeros(rows * k + 16, dtype=torch.int8, device="cuda")
        v = flat[off:off + rows * k].view(rows, k)
        v.copy_(torch.randint(-127, 128, (rows, k), generator=g, device="cuda"))
        return v
    x, w, wu = codes(m), codes(n), codes(n)
    x[1] = 0  # sums of 0: 0 whatever the scales
    for sx, sw in ((1e-30, 1e-12), (1e22, 1e20)):
        xs, ws = torch.full((m,), sx, device="cuda"), torch.full((n,), sw, device="cuda")
        one = torch.full((n,), 1 / sx, device="cuda")  # the gate's scales undone
        if sx > 1:
            x[2:] = 0
        y = torch.full((m, n), float("nan"), device="cuda")
        up = dict(w_up=wu.data_ptr(), w_up_scale=one.data_ptr()) if gated else {}
        api.linear(m, n, k, DT["i8"], x.data_ptr(), w.data_ptr(), y.data_ptr(), DT["f32"], x_scale=xs.data_ptr(),
                   w_scale=ws.data_ptr(), activation=api.ACTIVATIONS["none"], **up)
        rows = slice(None) if sx < 1 else slice(1, None)
        want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
        u = torch.ones_like(want)
        if gated:
            u = (x.double() @ wu.double().T) * xs.double()[:, None] * one.double()
        want = want * u
        # three products of f32 for each factor, on sums that f32 holds exactly; the first may be subnormal
        bound = 2.0 ** -21 * want.abs() + 2.0 ** -149 * (1 + u.abs())
        assert ((y.double() - want).abs() <= bound)[rows].all()
