"""The 8-bit operators on the GPU against their definition in 64 bits (oracle/fp8_ref.py).

Tolerances, derived before the first run.  Packing is exact: bytes and restored values are compared for equality.  A product's
operands are then known exactly, and what is left is the fp32 summation and one rounding of the result.  With S = sum |x||w| (+ the
other terms' magnitudes), a sum of K products in fp32 is off by at most K * 2^-24 * S for any order of additions rounded to nearest
(each of K additions is off by half a step of a partial sum, at most S); the matrix pipe may cut rather than round while it
aligns terms, which doubles that: (K + 4) * 2^-23 * S.  Rounding to bf16 adds 2^-8 of the result (half a step is eps / 2).

Results in bf16 come from the 8-bit matrix instruction, which adds eight consecutive products on one exponent: with 2^E at most the
largest of the eight magnitudes, every other product is cut to a multiple of 2^(E-13), so the seven lose less than
7 * 2^-13 * largest.  Summed over the eights that is 7 * 2^-13 * G, G = sum over eights of the largest |x||w|.  (Measured on the
instruction: a product of 2^-14 of its neighbour vanishes, one of 2^-13 stays, one eight positions away stays to 2^-23.)
"""
import math

import pytest
import torch

from oracle import fp8_ref as R

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _rand(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * scale


def _bytes(t):
    return t.cpu().view(torch.uint8)


def _same(a, b):
    """Equal, a NaN of either sign equal to a NaN."""
    a, b = a.double(), b.double()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0, 9e99, -9e99),
                                                                       torch.nan_to_num(b, 0.0, 9e99, -9e99))


def _eights(a, b):
    """G of the head of the file for a (rows, K) . b (n, K)^T."""
    a, b = a.abs(), b.abs()
    g = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64)
    for k in range(0, a.shape[1], 8):
        g += (a[:, None, k:k + 8] * b[None, :, k:k + 8]).amax(-1)
    return g


def _close(got, want, size, terms, dtype, eights=0.0):
    """Elementwise within the bound at the head of the file; `size` is S, `terms` the number of added products, `eights` G."""
    got = got.double().cpu()
    tol = (terms + 4) * 2.0 ** -23 * size
    if dtype == torch.bfloat16:
        tol = tol + 7 * 2.0 ** -13 * eights
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -133
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outside, worst {float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.3f} of the bound"


DTYPES = [torch.bfloat16, torch.float32]


# ------------------------------------------------------------------ packing
def _awkward(rows, c, dtype, seed):
    x = _rand((rows, c), seed) * torch.exp(3 * _rand((rows, 1), seed + 1))
    if rows > 4:
        x[0] = 0.0
        x[1] *= 1e-36                       # the scale's exponent reaches its floor
        x[2] = torch.exp(18 * _rand((c,), seed + 2))
        x[3, 0] = 3.0e38
        x[4, c // 2] = float("nan")
        if rows > 6:
            x[5, 0], x[5, c - 1] = float("inf"), -float("inf")
            x[6] = float("-inf")
    return x.to(dtype)


PACK_SHAPES = [(1, 1), (1, 8), (3, 17), (9, 128), (8, 129), (7, 250), (33, 1001), (2, 2500), (70, 16), (300, 3), (16, 384)]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,c", PACK_SHAPES)
def test_pack_and_unpack(dev, rows, c, dt, fmt):
    from mad_amd import ops
    x = _awkward(rows, c, dt, 10 * rows + c)
    values, ex = R.pack_rows(x, fmt)
    q, s = R.stored(values, ex, fmt)
    p = ops.pack_fp8(x.to(dev), fmt)
    assert p.q.dtype == R.TYPE[fmt] and p.shape == (rows, c) and p.dtype == dt
    assert torch.equal(_bytes(p.scale), s)
    assert _same(p.q.float().cpu(), q.view(R.TYPE[fmt]).float())
    assert torch.equal(_bytes(p.q) * 0 + _bytes(p.q), _bytes(p.q)) and not bool(_bytes(p.q)[:, c:].any())
    back = ops.unpack_fp8(p)
    assert back.dtype == dt and tuple(back.shape) == (rows, c)
    assert _same(back.cpu(), values.to(torch.float32).to(dt))


def test_pack_keeps_leading_axes_and_takes_no_rows(dev):
    from mad_amd import ops
    x = _rand((2, 3, 5, 40), 1).to(torch.bfloat16).to(dev)
    p = ops.pack_fp8(x)
    flat = ops.pack_fp8(x.view(30, 40))
    assert torch.equal(_bytes(p.q), _bytes(flat.q)) and torch.equal(ops.unpack_fp8(p).view(30, 40), ops.unpack_fp8(flat))
    y = ops.linear_fp8(x[0, 0, 0, :].contiguous(), ops.pack_weight_fp8(_rand((24, 40), 2).to(dev)))
    assert tuple(y.shape) == (24,)
    one = ops.pack_fp8(x[0, 0, 0, :].contiguous())
    assert torch.equal(_bytes(one.q)[0, :40], _bytes(flat.q)[0, :40])
    e = ops.pack_fp8(torch.empty((0, 40), device=dev))
    assert tuple(ops.unpack_fp8(e).shape) == (0, 40)


def test_pack_of_an_unaligned_view(dev):
    """Rows of odd length, and a tensor that starts anywhere: elements are only aligned to their own size."""
    from mad_amd import ops
    for dt in DTYPES:
        buf = _rand((1 + 11 * 131,), 3).to(dt).to(dev)
        view = buf[1:].view(11, 131)
        values, _ = R.pack_rows(view.cpu())
        assert torch.equal(ops.unpack_fp8(ops.pack_fp8(view)).cpu().double(), values)


def test_pack_writes_nothing_behind_the_last_row(dev):
    from mad_amd import _lib, ops
    rows, c = 5, 200
    x = _rand((rows, c), 5).to(dev)
    q = torch.full((rows + 3, 208), 0xAB, dtype=torch.uint8, device=dev)
    s = torch.full((rows + 3, 4), 0xAB, dtype=torch.uint8, device=dev)
    st = torch.cuda.current_stream().cuda_stream
    ops.check(_lib.lib.mad_pack_fp8(x.data_ptr(), _lib.MAD_F32, _lib.MAD_E4M3, rows, c, q.data_ptr(), s.data_ptr(), st), "pack")
    out = torch.full((rows + 3, c), 7.0, device=dev)
    ops.check(_lib.lib.mad_unpack_fp8(q.data_ptr(), s.data_ptr(), _lib.MAD_E4M3, rows, c, out.data_ptr(), _lib.MAD_F32, st), "unpack")
    assert bool((q[rows:] == 0xAB).all()) and bool((s[rows:] == 0xAB).all()) and bool((out[rows:] == 7.0).all())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (70, 300), (520, 40), (256, 640)])
def test_pack_weight(dev, n, k, dt):
    from mad_amd import ops
    w = (_rand((n, k), n + k) * torch.exp(2 * _rand((n, 1), 2))).to(dt)
    if n > 130:
        w[129:] = 0.0                       # blocks without a magnitude
    values, ex = R.pack_weight(w)
    q, s = R.stored(values, ex, rows_per_scale=128)
    qt, st = R.stored(values.t().contiguous(), ex.t().contiguous(), rows_per_scale=128)
    p = ops.pack_weight_fp8(w.to(dev), transposed=True)
    zero = lambda t: torch.where(t == 0x80, 0, t)          # the oracle does not keep the sign of a zero
    assert torch.equal(zero(_bytes(p.q)), zero(q)) and torch.equal(_bytes(p.scale), s)
    assert torch.equal(zero(_bytes(p.qt)), zero(qt)) and torch.equal(_bytes(p.scale_t), st)
    assert ops.pack_weight_fp8(w.to(dev)).qt is None


# ------------------------------------------------------------------ GroupNorm application with a checkpoint
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act,p", [(True, 0.0), (False, 0.0), (True, 0.25)])
@pytest.mark.parametrize("shape", [(2, 3, 5, 8), (1, 1, 1, 128), (3, 4, 4, 192), (2, 7, 9, 640), (1, 2, 2, 2304)])
def test_norm_save_and_restore(dev, shape, act, p, dt):
    from mad_amd import ops
    B, H, W, C = shape
    x = (_rand(shape, 1) * 1.7 + 0.3).to(dt).to(dev)
    coef = torch.stack((1 + 0.2 * _rand((B, C), 2), 0.3 * _rand((B, C), 3)), -1).contiguous().to(dev)
    y, x8 = ops.gn_apply_save(x, coef, act, drop_seed=77, drop_p=p)
    assert torch.equal(y, ops.gn_apply(x, coef, act, drop_seed=77, drop_p=p))
    ref = ops.pack_fp8(x)
    assert torch.equal(_bytes(x8.q), _bytes(ref.q)) and torch.equal(x8.scale, ref.scale)
    xr, yr = ops.gn_apply_restore(x8, coef, act, drop_seed=77, drop_p=p)
    assert torch.equal(xr, ops.unpack_fp8(ref)) and xr.shape == x.shape
    assert torch.equal(yr, ops.gn_apply(xr, coef, act, drop_seed=77, drop_p=p))


def test_norm_takes_no_images(dev):
    from mad_amd import ops
    y, p = ops.gn_apply_save(torch.empty((0, 4, 4, 64), device=dev), torch.empty((0, 64, 2), device=dev), True)
    x, y2 = ops.gn_apply_restore(p, torch.empty((0, 64, 2), device=dev), True)
    assert y.numel() == x.numel() == y2.numel() == 0


# ------------------------------------------------------------------ products
LINEAR = [
    # rows, K, N
    (1, 128, 16), (1, 768, 768), (1, 1, 1), (2, 17, 5), (16, 256, 64), (17, 200, 33), (31, 1000, 130), (33, 640, 384),
    (64, 384, 1152), (65, 128, 128), (100, 130, 250), (130, 48, 260), (257, 272, 513), (300, 2048, 96), (513, 384, 256), (1, 5000, 40),
]


def _linear_case(rows, k, n, dt, dev, seed=0):
    x = (_rand((rows, k), seed + 1) * torch.exp(0.5 * _rand((k,), seed + 2))).to(dt)
    w = _rand((n, k), seed + 3, 1 / math.sqrt(k))
    bias = _rand((n,), seed + 4, 0.1)
    res = _rand((rows, n), seed + 5).to(dt)
    return x, w, bias, res


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k,n", LINEAR)
def test_linear(dev, rows, k, n, dt):
    from mad_amd import ops
    x, w, bias, res = _linear_case(rows, k, n, dt, dev)
    xv, wv = R.pack_rows(x)[0], R.pack_weight(w)[0]
    plain, size, g8 = xv @ wv.t(), xv.abs() @ wv.abs().t(), _eights(xv, wv)
    pw = ops.pack_weight_fp8(w.to(dev))
    y = ops.linear_fp8(x.to(dev), pw)
    assert y.dtype == dt and tuple(y.shape) == (rows, n)
    _close(y, plain, size, k, dt, g8)
    # from the packed input: another launch of the same product
    x8 = ops.pack_fp8(x.to(dev))
    _close(ops.linear_fp8(x8, pw), plain, size, k, dt, g8)
    want = plain + bias.double() + res.double()
    full = size + bias.double().abs() + res.double().abs()
    y, saved = ops.linear_fp8(x.to(dev), pw, bias=bias.to(dev), residual=res.to(dev), save=True)
    _close(y, want, full, k, dt, g8)
    assert torch.equal(_bytes(saved.q), _bytes(x8.q)) and torch.equal(saved.scale, x8.scale)
    assert torch.equal(ops.linear_fp8(saved, pw, bias=bias.to(dev), residual=res.to(dev)), y)


@pytest.mark.parametrize("rows,k,n", [(1, 300, 20), (40, 256, 128), (200, 300, 130), (300, 512, 256)])
def test_linear_of_the_wide_range_type(dev, rows, k, n):
    from mad_amd import ops
    for dt in DTYPES:
        x, w, bias, _ = _linear_case(rows, k, n, dt, dev, 40)
        xv, wv = R.pack_rows(x, "e5m2")[0], R.pack_weight(w)[0]
        y = ops.linear_fp8(ops.pack_fp8(x.to(dev), "e5m2"), ops.pack_weight_fp8(w.to(dev)), bias=bias.to(dev))
        _close(y, xv @ wv.t() + bias.double(), xv.abs() @ wv.abs().t() + bias.double().abs(), k, dt, _eights(xv, wv))


# Sizes that fill the chip with tiles (128 x 128 and 256 x 256), ragged in every direction: rows, K, N.  The operands' values are the
# packed ones restored on the GPU (compared with the oracle above); product and bounds in fp64 on the GPU, in slices.
LARGE = [(4100, 272, 1000), (8200, 200, 2050), (33000, 640, 264), (2100, 130, 4100), (16400, 384, 1152), (65, 16, 33000), (70000, 100, 130),
         (8192, 1152, 2048), (5000, 17, 2303)]


def _large_check(got, x, w, extra, extra_size, terms, dtype):
    for lo in range(0, got.shape[0], 1024):
        a = x[lo:lo + 1024].double()
        want, size = a @ w.t(), a.abs() @ w.abs().t()
        g8 = torch.zeros_like(want)
        if dtype == torch.bfloat16:
            for k in range(0, w.shape[1], 8):
                top = torch.zeros_like(want)
                for j in range(k, min(k + 8, w.shape[1])):
                    top = torch.maximum(top, a[:, j, None].abs() * w[None, :, j].abs())
                g8 += top
        if extra is not None:
            want, size = want + extra[lo:lo + 1024], size + extra_size[lo:lo + 1024]
        tol = (terms + 4) * 2.0 ** -23 * size
        if dtype == torch.bfloat16:
            tol = (tol + 7 * 2.0 ** -13 * g8) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -133
        assert bool(((got[lo:lo + 1024].double() - want).abs() <= tol).all()), f"rows from {lo}"


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k,n", LARGE)
def test_linear_over_many_tiles(dev, rows, k, n, dt):
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(rows + k + n)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)
    x8 = ops.pack_fp8((rand(rows, k) * torch.exp(0.5 * rand(k))).to(dt), "e5m2" if n % 2 else "e4m3")
    w = rand(n, k) / math.sqrt(k)
    pw = ops.pack_weight_fp8(w, transposed=True)
    xv = ops.unpack_fp8(x8)
    eye = ops.pack_fp8(torch.eye(k, device=dev))
    wv = ops.linear_fp8(eye, pw).t().double()               # the weight's values: products with 1 and 0 alone are exact
    _large_check(ops.linear_fp8(x8, pw), xv, wv, None, None, k, dt)
    bias, res = rand(n), rand(rows, n).to(dt)
    got = ops.linear_fp8(x8, pw, bias=bias, residual=res)
    _large_check(got, xv, wv, bias.double() + res.double(), bias.double().abs() + res.double().abs(), k, dt)
    # nothing behind the last row is written
    buf = torch.full((rows + 2, n), 7.0, dtype=dt, device=dev)
    from mad_amd import _lib
    ops.check(_lib.lib.mad_linear_fp8(x8.q.data_ptr(), ops._FP8_CODES[x8.q.dtype], x8.scale.data_ptr(), pw.q.data_ptr(), pw.scale.data_ptr(),
                                      bias.data_ptr(), res.data_ptr(), buf.data_ptr(), ops._dtype_code(buf), rows, k, n,
                                      torch.cuda.current_stream().cuda_stream), "mad_linear_fp8")
    assert torch.equal(buf[:rows], got) and bool((buf[rows:] == 7.0).all())


# bf16 inputs long enough for the form that rounds them on the way in, of one to four blocks, whole and partial, and around its limits
ROWS_FORM = [(33000, 64, 200), (32768, 128, 128), (32769, 136, 513), (40001, 256, 768), (33333, 384, 66), (65600, 392, 384), (33000, 512, 2048),
             (33000, 512, 2056), (33000, 520, 64), (33000, 60, 64)]


# ... of five to nine blocks, where a unit holds one workgroup
ROWS_FORM += [(32768, 640, 72), (32700, 1152, 200), (65500, 776, 130), (32768, 1024, 2048), (65536, 904, 66), (32768, 1160, 64), (45000, 1152, 96)]


@pytest.mark.parametrize("rows,k,n", ROWS_FORM)
def test_one_launch_is_packing_and_product(dev, rows, k, n):
    """The rounded x, if wanted, and y are those of the two calls, bit for bit; rows that are not finite included."""
    from mad_amd import _lib, ops
    g = torch.Generator(device=dev).manual_seed(rows + k + n)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)
    x = (rand(rows, k) * torch.exp(2 * rand(rows, 1))).to(torch.bfloat16)
    x[1, 3], x[5] = float("nan"), 0.0
    x[rows - 1, k // 2], x[7] = float("inf"), float("-inf")
    x[9] *= 2.0 ** -120
    pw = ops.pack_weight_fp8(rand(n, k) / math.sqrt(k))
    bias, res = rand(n), rand(rows, n).to(torch.bfloat16)
    x8 = ops.pack_fp8(x)
    for b, r in ((None, None), (bias, res)):
        want = ops.linear_fp8(x8, pw, bias=b, residual=r)
        y = ops.linear_fp8(x, pw, bias=b, residual=r)
        ys, kept = ops.linear_fp8(x, pw, bias=b, residual=r, save=True)
        assert _same(y, want) and _same(ys, want)
        assert _same(kept.q.float(), x8.q.float()) and torch.equal(kept.scale, x8.scale)
        assert not bool(_bytes(kept.q)[:, k:].any())
    buf = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device=dev)
    q, s = torch.full((rows + 2, x8.q.shape[1]), 0x11, dtype=torch.uint8, device=dev), torch.full((rows + 2, x8.scale.shape[1]), 0x11, dtype=torch.uint8, device=dev)
    ops.check(_lib.lib.mad_linear_fp8_save(x.data_ptr(), _lib.MAD_BF16, _lib.MAD_E4M3, pw.q.data_ptr(), pw.scale.data_ptr(), bias.data_ptr(),
                                           res.data_ptr(), buf.data_ptr(), q.data_ptr(), s.data_ptr(), rows, k, n,
                                           torch.cuda.current_stream().cuda_stream), "mad_linear_fp8_save")
    assert _same(buf[:rows], want) and bool((buf[rows:] == 7.0).all()) and bool((q[rows:] == 0x11).all()) and bool((s[rows:] == 0x11).all())


# sizes around the limits of the form that rounds x inside a small product: rows, K, N
SMALL_SAVE = [(1, 1, 1), (1, 1000, 70), (16, 272, 4200), (31, 130, 33), (32, 520, 40), (33, 128, 16), (64, 1001, 328), (777, 200, 137), (1000, 384, 500),
              (512, 1024, 640), (20, 4097, 64), (2048, 96, 328), (777, 1000, 1024)]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k,n", SMALL_SAVE)
def test_packed_inside_a_small_product(dev, rows, k, n, dt, fmt):
    """The kept x is that of packing alone and y that of the kept x, bit for bit; nothing behind either is written, and y without
    keeping x holds the product's bound."""
    from mad_amd import _lib, ops
    x, w, bias, res = (t.to(dev) for t in _linear_case(rows, k, n, dt, dev, 60))
    if rows > 8:
        x[3, k // 2], x[5, 0], x[6] = float("nan"), float("inf"), 0.0
        x[7] *= 2.0 ** -120
    pw = ops.pack_weight_fp8(w)
    x8 = ops.pack_fp8(x, fmt)
    stored = {"e4m3": _lib.MAD_E4M3, "e5m2": _lib.MAD_E5M2}[fmt]
    for b, r in ((None, None), (bias, res)):
        want = ops.linear_fp8(x8, pw, bias=b, residual=r)
        y = torch.full((rows + 2, n), 7.0, dtype=dt, device=dev)
        q, s = (torch.full((rows + 2, t.shape[1]), 0x11, dtype=torch.uint8, device=dev) for t in (x8.q, x8.scale))
        ops.check(_lib.lib.mad_linear_fp8_save(x.data_ptr(), ops._dtype_code(x), stored, pw.q.data_ptr(), pw.scale.data_ptr(),
                                               None if b is None else b.data_ptr(), None if r is None else r.data_ptr(), y.data_ptr(),
                                               q.data_ptr(), s.data_ptr(), rows, k, n, torch.cuda.current_stream().cuda_stream), "mad_linear_fp8_save")
        assert _same(q[:rows].view(x8.q.dtype).float(), x8.q.float()) and torch.equal(s[:rows], x8.scale) and not bool(q[:rows, k:].any())
        assert _same(y[:rows], want)
        assert bool((y[rows:] == 7.0).all()) and bool((q[rows:] == 0x11).all()) and bool((s[rows:] == 0x11).all())
    if fmt == "e4m3":
        ok = [i for i in range(rows) if i not in (3, 5)]
        xv, wv = R.pack_rows(x.cpu()[ok])[0], R.pack_weight(w.cpu())[0]
        _close(ops.linear_fp8(x, pw)[ok], xv @ wv.t(), xv.abs() @ wv.abs().t(), k, dt, _eights(xv, wv))


@pytest.mark.parametrize("rows", [3, 300])
def test_rows_do_not_touch_each_other(dev, rows):
    """NaN and infinities in one row reach that row of y alone, and zero rows give the bias."""
    from mad_amd import ops
    k, n = 320, 144
    x, w, bias, _ = _linear_case(rows, k, n, torch.float32, dev, 9)
    pw = ops.pack_weight_fp8(w.to(dev))
    clean = ops.linear_fp8(x.to(dev), pw, bias=bias.to(dev))
    x[1, 5], x[1, 200] = float("nan"), float("inf")
    x[2] = 0.0
    y = ops.linear_fp8(x.to(dev), pw, bias=bias.to(dev))
    assert bool(torch.isnan(y[1]).all()) and torch.equal(y[2].cpu(), bias)
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


def test_scales_far_apart(dev):
    """Blocks of very different size in one row, down to the floor of the exponents: each product keeps its own scale."""
    from mad_amd import ops
    for rows in (2, 130):
        for dt in DTYPES:
            x = _rand((rows, 512), 3)
            x[:, 128:256] *= 2.0 ** -60
            x[:, 256:384] *= 2.0 ** 60
            w = _rand((64, 512), 4)
            w[:, 128:256] *= 2.0 ** 70
            w[:, 256:384] *= 2.0 ** -50
            x = x.to(dt)
            xv, wv = R.pack_rows(x)[0], R.pack_weight(w)[0]
            y = ops.linear_fp8(x.to(dev), ops.pack_weight_fp8(w.to(dev)))
            _close(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), 512, dt, _eights(xv, wv))


@pytest.mark.parametrize("rows", [2, 70, 5000, 33000])
def test_weights_that_are_not_finite(dev, rows):
    """A NaN or an infinity of the weight makes its column of y NaN and no other."""
    from mad_amd import ops
    k, n = 200, 300
    g = torch.Generator(device=dev).manual_seed(4)
    w = torch.randn((n, k), generator=g, device=dev)
    x = torch.randn((rows, k), generator=g, device=dev).to(torch.bfloat16)
    clean = ops.linear_fp8(x, ops.pack_weight_fp8(w))
    w[7, 3], w[200, 199] = float("nan"), float("inf")
    y = ops.linear_fp8(x, ops.pack_weight_fp8(w))
    keep = [i for i in range(n) if i not in (7, 200)]
    assert torch.equal(y[:, keep], clean[:, keep]) and bool(torch.isnan(y[:, [7, 200]]).all())


def test_values_at_the_floor_of_the_exponents(dev):
    """Activations whose scale is the smallest there is (their values are subnormal in bf16): products and gradients keep them."""
    from mad_amd import ops
    for dt in DTYPES:
        x = (_rand((96, 256), 1) * 2.0 ** -124).to(dt)
        x8 = ops.pack_fp8(x.to(dev))
        assert bool((x8.scale[:, :2] == 1).all())
        xv = R.pack_rows(x)[0]
        assert _same(ops.unpack_fp8(x8).cpu(), xv.float().to(dt))
        w = _rand((48, 256), 2) * 2.0 ** 60
        wv = R.pack_weight(w)[0]
        _close(ops.linear_fp8(x8, ops.pack_weight_fp8(w.to(dev))), xv @ wv.t(), xv.abs() @ wv.abs().t(), 256, dt, _eights(xv, wv))
        dy = (_rand((96, 64), 3) * 2.0 ** 60).to(dt)
        _, dw, _ = ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False)
        # the gradient takes x in bf16: 2^-126 times an 8-bit value may lie between two multiples of 2^-133, bf16's smallest step, and is
        # then off by at most half of it, so dw by at most 2^-134 * sum |dy|, added to S as (sum |dy| * 2^-134) / (100 * 2^-23)
        size = dy.double().abs().t() @ xv.abs() + dy.double().abs().sum(0)[:, None] * (2.0 ** -134 / (100 * 2.0 ** -23))
        _close(dw, dy.double().t() @ xv, size, 96, torch.float32)


def test_linear_of_unaligned_operands(dev):
    """A bias, a residual and an input that start at any element."""
    from mad_amd import ops
    for dt in DTYPES:
        for rows in (5, 200):
            x, w, bias, res = _linear_case(rows, 96, 64, dt, dev, 21)
            off = lambda t: torch.cat([t.flatten()[:1], t.flatten()]).to(dev)[1:].view(t.shape)
            pw = ops.pack_weight_fp8(w.to(dev))
            a = ops.linear_fp8(x.to(dev), pw, bias=bias.to(dev), residual=res.to(dev))
            assert torch.equal(ops.linear_fp8(off(x), pw, bias=off(bias), residual=off(res)), a)


def test_linear_keeps_leading_axes_and_takes_no_rows(dev):
    from mad_amd import ops
    x, w, bias, _ = _linear_case(24, 96, 40, torch.bfloat16, dev, 3)
    pw = ops.pack_weight_fp8(w.to(dev), transposed=True)
    y = ops.linear_fp8(x.to(dev).view(2, 3, 4, 96), pw)
    assert tuple(y.shape) == (2, 3, 4, 40) and torch.equal(y.view(24, 40), ops.linear_fp8(x.to(dev), pw))
    y, x8 = ops.linear_fp8(x.to(dev)[:0], pw, bias=bias.to(dev), save=True)
    assert tuple(y.shape) == (0, 40)
    dw, db = torch.ones((40, 96), device=dev), torch.ones((40,), device=dev)
    dx, _, _ = ops.linear_fp8_backward(y, x8, pw, dw=dw, dbias=db, accumulate=True)
    assert tuple(dx.shape) == (0, 96) and bool((dw == 1).all()) and bool((db == 1).all())
    _, dw, db = ops.linear_fp8_backward(y, x8, pw)
    assert not bool(dw.any()) and not bool(db.any())


def test_refusals_on_the_gpu(dev):
    from mad_amd import ops
    x, w, bias, res = _linear_case(8, 96, 40, torch.bfloat16, dev, 3)
    x, pw = x.to(dev), ops.pack_weight_fp8(w.to(dev))
    with pytest.raises(ValueError, match="columns"):
        ops.linear_fp8(x[:, :64].contiguous(), pw)
    with pytest.raises(ValueError, match="contiguous"):
        ops.linear_fp8(x[:, ::2], pw)
    with pytest.raises(TypeError):
        ops.linear_fp8(x.half(), pw)
    with pytest.raises(ValueError, match="bias"):
        ops.linear_fp8(x, pw, bias=torch.zeros(41, device=dev))
    with pytest.raises(ValueError, match="residual"):
        ops.linear_fp8(x, pw, residual=torch.zeros((8, 41), device=dev, dtype=x.dtype))
    with pytest.raises(ValueError, match="residual"):
        ops.linear_fp8(x, pw, residual=torch.zeros((8, 40), device=dev))
    with pytest.raises(ValueError, match="8-bit type"):
        ops.pack_fp8(x, "e3m4")
    with pytest.raises(ValueError, match="columns"):
        ops.pack_fp8(torch.zeros((4, 0), device=dev))
    with pytest.raises(ValueError, match="matrix"):
        ops.pack_weight_fp8(torch.zeros(4, device=dev))
    y, x8 = ops.linear_fp8(x, pw, save=True)
    with pytest.raises(ValueError, match="transposed"):
        ops.linear_fp8_backward(y, x8, pw)
    with pytest.raises(ValueError, match="packed weight"):
        ops.linear_fp8_backward(y, x8)
    with pytest.raises(ValueError, match="does not belong"):
        ops.linear_fp8_backward(y.float(), x8, need_dx=False)
    with pytest.raises(ValueError, match="accumulate"):
        ops.linear_fp8_backward(y, x8, need_dx=False, accumulate=True)
    with pytest.raises(ValueError, match="dw must"):
        ops.linear_fp8_backward(y, x8, need_dx=False, dw=torch.zeros((40, 95), device=dev))
    with pytest.raises(ValueError, match="do not belong"):
        ops.unpack_fp8(x8._replace(shape=(9, 96)))
    with pytest.raises(TypeError, match="e4m3"):
        ops.gn_apply_restore(ops.pack_fp8(x.view(1, 2, 4, 96), "e5m2"), torch.zeros((1, 96, 2), device=dev), True)
    with pytest.raises(ValueError, match="coef"):
        ops.gn_apply_save(x.view(1, 2, 4, 96), torch.zeros((1, 95, 2), device=dev), True)


def test_refusals_of_what_is_not_packed(dev):
    from mad_amd import ops
    x, w, _, _ = _linear_case(8, 96, 40, torch.bfloat16, dev, 3)
    x, w = x.to(dev), w.to(dev)
    pw = ops.pack_weight_fp8(w, transposed=True)
    y, x8 = ops.linear_fp8(x, pw, save=True)
    for call in (lambda: ops.linear_fp8(x, w), lambda: ops.unpack_fp8(x), lambda: ops.linear_fp8_backward(y, x, pw),
                 lambda: ops.gn_apply_restore(x.view(1, 2, 4, 96), torch.zeros((1, 96, 2), device=dev), True)):
        with pytest.raises(TypeError, match="pack_weight_fp8|Fp8Tensor"):
            call()
    with pytest.raises(ValueError, match="packed weight"):
        ops.linear_fp8_backward(y, x8, w)


# ------------------------------------------------------------------ gradients
BACKWARD = [(1, 16, 8), (5, 200, 137), (64, 128, 128), (300, 96, 260), (700, 384, 130), (1500, 130, 70), (2100, 256, 384)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,k,n", BACKWARD)
def test_linear_backward(dev, rows, k, n, fmt, dt):
    from mad_amd import ops
    x, w, _, _ = _linear_case(rows, k, n, dt, dev, 60)
    dy = (1e-3 * _rand((rows, n), 7) * torch.exp(_rand((rows, 1), 8))).to(dt)
    xv, wv, gv, g = R.pack_rows(x)[0], R.pack_weight(w)[0], R.pack_rows(dy, fmt)[0], dy.double()
    pw = ops.pack_weight_fp8(w.to(dev), transposed=True)
    x8 = ops.pack_fp8(x.to(dev))
    dx, dw, db = ops.linear_fp8_backward(dy.to(dev), x8, pw, grad_fmt=fmt)
    assert dx.dtype == dt and dx.shape == x.shape and dw.dtype == db.dtype == torch.float32
    _close(dx, gv @ wv, gv.abs() @ wv.abs(), n, dt, _eights(gv, wv.t()))
    _close(dw, g.t() @ xv, g.abs().t() @ xv.abs(), rows, torch.float32)
    _close(db, g.sum(0), g.abs().sum(0), rows, torch.float32)
    # added to what is there; nothing but dw asked for
    base_w, base_b = torch.full((n, k), 0.5, device=dev), torch.full((n,), 0.25, device=dev)
    ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False, dw=base_w, dbias=base_b, accumulate=True)
    _close(base_w, g.t() @ xv + 0.5, g.abs().t() @ xv.abs() + 0.5, rows, torch.float32)
    _close(base_b, g.sum(0) + 0.25, g.abs().sum(0) + 0.25, rows, torch.float32)
    none, dw2, nodb = ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False, need_dbias=False)
    assert none is None and nodb is None and torch.equal(dw2, dw)


# rows, K, N: many shares of the rows, tiles of 128 and of 256, ragged in every direction, rows of dy that are no whole 16 bytes
WGRAD_LARGE = [(66000, 272, 136), (333, 4000, 4104), (20001, 384, 1152), (5000, 16, 8), (3000, 1040, 131), (64, 4096, 4096), (129, 130, 264),
               (30000, 768, 2304), (9000, 640, 520), (2000, 1152, 1536), (40000, 200, 1152)]


# as many tiles as units and rows enough that the bias gradient is shared over them: one share, and its parts joined alone
WGRAD_LARGE += [(5000, 4096, 4112), (4001, 4100, 4095)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k,n", WGRAD_LARGE)
def test_weight_gradient_over_many_tiles(dev, rows, k, n, dt):
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(rows + k + n)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)
    dy = (1e-3 * rand(rows, n) * torch.exp(rand(rows, 1))).to(dt)
    x8 = ops.pack_fp8((rand(rows, k) * torch.exp(2 * rand(rows, 1))).to(dt), "e5m2" if rows % 2 else "e4m3")
    xv, gd = ops.unpack_fp8(x8).double(), dy.double()
    _, dw, db = ops.linear_fp8_backward(dy, x8, need_dx=False)
    within = lambda got, want, size: bool(((got.double() - want).abs() <= (rows + 4) * 2.0 ** -23 * size).all())
    want, size = gd.t() @ xv, gd.abs().t() @ xv.abs()
    assert within(dw, want, size) and within(db, gd.sum(0), gd.abs().sum(0))
    again = ops.linear_fp8_backward(dy, x8, need_dx=False)
    assert torch.equal(again[1], dw) and torch.equal(again[2], db)
    base, bb = torch.full((n + 1, k), 0.5, device=dev), torch.full((n + 1,), 0.25, device=dev)
    ops.linear_fp8_backward(dy, x8, need_dx=False, dw=base[:n], dbias=bb[:n], accumulate=True)
    assert within(base[:n], want + 0.5, size + 0.5) and within(bb[:n], gd.sum(0) + 0.25, gd.abs().sum(0) + 0.25)
    assert bool((base[n] == 0.5).all()) and float(bb[n]) == 0.25
    # dy anywhere in memory: the form that does not need whole pieces
    off = torch.cat([dy.flatten()[:1], dy.flatten()])[1:].view(rows, n)
    _, dw, db = ops.linear_fp8_backward(off, x8, need_dx=False)
    assert within(dw, want, size) and within(db, gd.sum(0), gd.abs().sum(0))


@pytest.mark.parametrize("dt", DTYPES)
def test_gradients_against_differences(dev, dt):
    """On small whole numbers every rounding of the operator is exact, so <g, y> is linear in x, w and the bias and differences of it
    over whole steps ARE its gradients' inner products with the steps."""
    from mad_amd import ops
    rows, k, n = 150, 140, 70
    gen = torch.Generator().manual_seed(5)
    ints = lambda *s: torch.randint(-3, 4, s, generator=gen).float()
    x, w, b, g = ints(rows, k), ints(n, k), ints(n), ints(rows, n)
    ex, ew, eb = ints(rows, k), ints(n, k), ints(n)

    def value(x, w, b):
        y = ops.linear_fp8(x.to(dev), ops.pack_weight_fp8(w.to(dev)), bias=b.to(dev))
        return float((y.double().cpu() * g.double()).sum())
    x8 = ops.pack_fp8(x.to(dt).to(dev))
    dx, dw, db = ops.linear_fp8_backward(g.to(dt).to(dev), x8, ops.pack_weight_fp8(w.to(dev), transposed=True))
    v = value(x, w, b)
    inner = lambda a, e: float((a.double().cpu() * e.double()).sum())
    # dx is a whole number of at most 9 * 70 = 630 in magnitude: bf16 holds it to half a step of 2^(9-7), i.e. 2
    slack = 2.0 * float(ex.abs().sum()) if dt == torch.bfloat16 else 0.0
    assert abs(value(x + ex, w, b) - v - inner(dx, ex)) <= slack
    assert value(x, w + ew, b) - v == inner(dw, ew)
    assert value(x, w, b + eb) - v == inner(db, eb)


def test_gradient_of_infinities(dev):
    """A gradient row that is not finite makes what it reaches NaN or infinite and nothing else."""
    from mad_amd import ops
    for dt in DTYPES:
        x8 = ops.pack_fp8(_rand((40, 64), 1).to(dt).to(dev))
        dy = _rand((40, 32), 2).to(dt)
        _, clean, cb = ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False)
        dy[3, 5], dy[9, 6] = float("inf"), float("nan")
        _, dw, db = ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False)
        keep = [i for i in range(32) if i not in (5, 6)]
        assert torch.equal(dw[keep], clean[keep]) and torch.equal(db[keep], cb[keep])
        assert not bool(torch.isfinite(dw[5:7]).any()) and bool(torch.isinf(db[5])) and bool(torch.isnan(db[6]))


# ------------------------------------------------------------------ as they are used
def _chain(ops, x, coef, w, bias, dy, res):
    """Forward of a projection after a norm with its checkpoint, then its backward from the checkpoint."""
    pw = ops.pack_weight_fp8(w, transposed=True)
    h, x8 = ops.gn_apply_save(x, coef, True, drop_seed=5, drop_p=0.1)
    y, h8 = ops.linear_fp8(h, pw, bias=bias, residual=res, save=True)
    xr, hr = ops.gn_apply_restore(x8, coef, True, drop_seed=5, drop_p=0.1)
    dh, dw, db = ops.linear_fp8_backward(dy, h8, pw)
    return y, xr, hr, dh, dw, db


def _chain_inputs(dev, seed, dt=torch.bfloat16):
    B, H, W, C, N = 3, 8, 16, 192, 320
    return ((_rand((B, H, W, C), seed) + 0.2).to(dt).to(dev), torch.stack((1 + 0.1 * _rand((B, C), 2), 0.1 * _rand((B, C), 3)), -1).contiguous().to(dev),
            _rand((N, C), 4, C ** -0.5).to(dev), _rand((N,), 5).to(dev), _rand((B, H, W, N), seed + 6, 1e-3).to(dt).to(dev),
            _rand((B, H, W, N), seed + 7).to(dt).to(dev))


def test_chain_is_deterministic_and_independent_of_the_stream(dev):
    from mad_amd import ops
    args = _chain_inputs(dev, 1)
    a = _chain(ops, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _chain(ops, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams share nothing."""
    from mad_amd import ops
    args = [_chain_inputs(dev, s) for s in (1, 30)]
    want = [_chain(ops, *a) for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_chain(ops, *args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(u, v) for u, v in zip(out, want[i]))


def test_chain_in_a_graph(dev):
    """Captured, replayed on new inputs with eager work between the replays: the eager results, bit for bit; two graphs captured
    after one another keep their own workspaces."""
    from mad_amd import ops
    bufs = [_chain_inputs(dev, 1), _chain_inputs(dev, 50)]
    graphs = []
    for args in bufs:
        _chain(ops, *args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _chain(ops, *args)
        graphs.append((g, out))
    for seed in (100, 200, 300):
        fresh = [_chain_inputs(dev, seed), _chain_inputs(dev, seed + 1)]
        for args, new in zip(bufs, fresh):
            for t, n in zip(args, new):
                t.copy_(n)
        for g, _ in graphs:
            g.replay()
        want = [_chain(ops, *new) for new in fresh]
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(u, v) for u, v in zip(out, w))


def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the rows at the far end are what they are in a small tensor."""
    from mad_amd import ops
    c = 128
    rows = (1 << 31) // c + 1000
    x = torch.zeros((rows, c), dtype=torch.bfloat16, device=dev)
    tail = _rand((1000, c), 3).to(torch.bfloat16).to(dev)
    x[-1000:] = tail
    p, small = ops.pack_fp8(x), ops.pack_fp8(tail)
    assert torch.equal(_bytes(p.q[-1000:]), _bytes(small.q)) and torch.equal(p.scale[-1000:], small.scale)
    assert torch.equal(ops.unpack_fp8(p)[-1000:], ops.unpack_fp8(small))
    pw = ops.pack_weight_fp8(_rand((16, c), 4).to(dev))
    assert torch.equal(ops.linear_fp8(p, pw)[-1000:], ops.linear_fp8(small, pw))
    coef = torch.ones((1, c, 2), device=dev)
    xr, y = ops.gn_apply_restore(p._replace(shape=(1, rows, 1, c)), coef, True)
    assert torch.equal(xr[0, -1000:, 0], ops.unpack_fp8(small))
    dy = torch.zeros((rows, 16), dtype=torch.bfloat16, device=dev)
    dy[-1000:] = _rand((1000, 16), 5).to(torch.bfloat16).to(dev)
    _, dw, _ = ops.linear_fp8_backward(dy, p, need_dx=False)
    g = dy[-1000:].double().cpu()
    xv = ops.unpack_fp8(small).double().cpu()
    # zero products add nothing; the order of the rest is one of 1000 terms and the shares' sums
    _close(dw, g.t() @ xv, g.abs().t() @ xv.abs(), 2000, torch.float32)
