"""The 8-bit operators at the limits of their operands: ends of allocations, share and step borders, the largest and smallest sizes
and values (GPU only).  Where operands are small whole numbers every product and sum is exact, so results are compared for equality;
other tolerances are derived beside the tests."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _at_the_end(t):
    """A copy of t whose last byte is the last one of an allocation of its own (whole 2 MiB pages, far above what a pool shares)."""
    n = t.numel() * t.element_size()
    page = 2 << 20
    buf = torch.empty(max(16 << 20, -(-n // page) * page), dtype=torch.uint8, device=t.device)
    view = buf[buf.numel() - n:].view(t.dtype).view(t.shape)
    view.copy_(t)
    return view


# rows, K, N: one to nine blocks, one share of the columns and two, last strips that are whole and that are not
@pytest.mark.parametrize("rows,k,n", [(32768, 64, 64), (33000, 136, 200), (40001, 256, 768), (33000, 512, 2048), (32768, 1152, 200)])
def test_rounding_product_with_weights_at_the_end_of_memory(dev, rows, k, n):
    """A long bf16 input is rounded inside the product, which copies the weights ahead in strips of 64 rows: nothing is asked for
    behind the last one, and y is that of weights that lie elsewhere."""
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(k)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)
    x = rand(rows, k).to(torch.bfloat16)
    w, bias = ops.pack_weight_fp8(rand(n, k) / math.sqrt(k)), rand(n)
    q = _at_the_end(w.q.view(torch.uint8)).view(w.q.dtype)
    edge = w._replace(q=q, scale=_at_the_end(w.scale))
    want = ops.linear_fp8(ops.pack_fp8(x), w, bias=bias)
    assert torch.equal(ops.linear_fp8(x, edge, bias=_at_the_end(bias)), want)
    assert torch.equal(ops.linear_fp8(x, edge, bias=bias, save=True)[0], want)


def test_norm_of_the_largest_image(dev):
    """2^31 - 1 pixels, the most that the entry point counts: the shares of the last workgroups end behind them."""
    from mad_amd import ops
    c, n, m = 8, (1 << 31) - 1, 1000
    torch.cuda.empty_cache()
    g = torch.Generator(device=dev).manual_seed(1)
    ends = [torch.randn((m, c), generator=g, device=dev).to(torch.bfloat16) for _ in range(2)]
    coef = torch.randn((1, c, 2), generator=g, device=dev)
    x = torch.zeros((1, n, 1, c), dtype=torch.bfloat16, device=dev)
    x[0, :m, 0], x[0, -m:, 0] = ends
    at = lambda t, i: (t[:m], t[-m:])[i]
    y, p = ops.gn_apply_save(x, coef, act=True)
    for i, e in enumerate(ends):
        want, small = ops.gn_apply_save(e.view(1, m, 1, c), coef, act=True)
        assert torch.equal(at(y[0], i), want[0])
        assert torch.equal(at(p.q, i).view(torch.uint8), small.q.view(torch.uint8)) and torch.equal(at(p.scale, i), small.scale)
    del x, y
    torch.cuda.empty_cache()
    xr, yr = ops.gn_apply_restore(p, coef, act=True)
    for i, e in enumerate(ends):
        x2, y2 = ops.gn_apply_restore(ops.pack_fp8(e.view(1, m, 1, c)), coef, act=True)
        assert torch.equal(at(xr[0], i), x2[0]) and torch.equal(at(yr[0], i), y2[0])
    del xr, yr, p
    torch.cuda.empty_cache()


def test_product_of_more_rows_than_one_launch_rounds(dev):
    """2^31 rows and some: the form that rounds 128 rows to a workgroup would count more threads than a launch holds."""
    from mad_amd import ops
    k, n, m = 8, 8, 1000
    torch.cuda.empty_cache()
    g = torch.Generator(device=dev).manual_seed(2)
    tail = torch.randn((m, k), generator=g, device=dev).to(torch.bfloat16)
    w = ops.pack_weight_fp8(torch.randn((n, k), generator=g, device=dev))
    x = torch.zeros(((1 << 31) + m, k), dtype=torch.bfloat16, device=dev)
    x[-m:] = tail
    y, x8 = ops.linear_fp8(x, w, save=True)
    del x
    small, t8 = ops.linear_fp8(tail, w, save=True)
    assert torch.equal(x8.q[-m:].view(torch.uint8), t8.q.view(torch.uint8)) and torch.equal(x8.scale[-m:], t8.scale)
    assert torch.equal(y[-m:], small) and not bool(y[:m].any())
    del y, x8
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [64, 61])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_gradients_near_the_smallest_numbers(dev, dt, n):
    """dy of 2^-136 to 2^-117.  bf16 enters the products as it is, fp32 in three bf16 terms cut toward zero to multiples of 2^-133.  The
    sums are whole numbers of the last place below 2^24 (300 * 2^12 * 8), so they are exact: dw and db are those of the cut dy."""
    from mad_amd import ops
    rows, k = 300, 96
    g = torch.Generator().manual_seed(n)
    x = torch.randint(-8, 9, (rows, k), generator=g).float() * 2.0 ** 60
    x8 = ops.pack_fp8(x.to(dt).to(dev))
    whole = torch.randint(1, 1 << 12, (rows, n), generator=g) * (2 * torch.randint(0, 2, (rows, n), generator=g) - 1)
    for e in (-136, -129):                                    # -129: nothing lies below 2^-133
        dy = (whole.double() * 2.0 ** e).float().to(dt)
        _, dw, db = ops.linear_fp8_backward(dy.to(dev), x8, need_dx=False)
        d = torch.trunc(dy.double() * 2.0 ** 133) * 2.0 ** -133
        assert torch.equal(d, dy.double()) == (e == -129 or dt == torch.bfloat16)
        assert torch.equal(dw.double().cpu(), d.t() @ x.double()) and torch.equal(db.double().cpu(), d.sum(0))


# rows, K, N of many shares, tiles of every size and ragged ends; one row, one step, one share and a row more
WGRAD = [(66000, 272, 136), (333, 4000, 4104), (20001, 384, 1152), (5000, 16, 8), (3000, 1040, 131), (64, 4096, 4096), (129, 130, 264),
         (30000, 768, 2304), (9000, 640, 520), (2000, 1152, 1536), (40000, 200, 1152), (5000, 4096, 4112), (4001, 4100, 4095),
         (1, 40, 24), (63, 384, 384), (65, 200, 520), (16384, 2048, 2048), (65536, 128, 384)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,n", WGRAD)
def test_weight_gradient_of_whole_numbers(dev, rows, k, n, dt):
    """Every sum is a whole number below 2^24 whatever the order of its additions, so dw and db are equal bit for bit in every form:
    a row, a step or a share that is lost, counted twice or scaled by its neighbour's scale shows.
    First in every row: |dy| <= 3, |x| <= 3 * 2^s with s = 0..3 by rows, at most 72 * 66000.  Then, in three rows of each column of dy,
    numbers of 22 bits (in fp32 all three terms of the split) against |x| <= 1: at most 3 * 2^22."""
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(rows + k + n)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g, device=dev)
    fmt = "e5m2" if rows % 2 else "e4m3"
    sparse = torch.zeros((rows, n), dtype=torch.int64, device=dev)
    for _ in range(min(3, rows)):
        sparse.scatter_(0, ints(0, rows - 1, 1, n), (2 * ints(0, (1 << 21) - 1, 1, n) + 1) * (2 * ints(0, 1, 1, n) - 1))
    size = 2.0 ** ints(0, 3, rows, 1).double()
    if dt == torch.bfloat16:
        sparse = sparse.clamp(-255, 255)                      # what eight bits hold
    for x, dy in ((ints(-3, 3, rows, k).double() * size, ints(-3, 3, rows, n)), (ints(-1, 1, rows, k).double(), sparse)):
        x8, dy = ops.pack_fp8(x.to(dt), fmt), dy.to(dt)
        want, want_b = dy.double().t() @ x, dy.double().sum(0)
        off = torch.cat([dy.flatten()[:1], dy.flatten()])[1:].view(rows, n)             # rows that start anywhere
        for d in (dy, off):
            _, dw, db = ops.linear_fp8_backward(d, x8, need_dx=False)
            assert torch.equal(dw.double(), want) and torch.equal(db.double(), want_b)
            dw, db = torch.full((n + 1, k), 5.0, device=dev), torch.full((n + 1,), -3.0, device=dev)
            ops.linear_fp8_backward(d, x8, need_dx=False, dw=dw[:n], dbias=db[:n], accumulate=True)
            assert torch.equal(dw[:n].double(), want + 5) and torch.equal(db[:n].double(), want_b - 3)
            assert bool((dw[n] == 5).all()) and float(db[n]) == -3


# rows, K, N of every form of the product: direct with 16, 32 and 64 rows, tiles of 128 and 256, rounding inside by 16 and by 128 rows
PRODUCT = [(1, 768, 768), (3, 4100, 40), (31, 1000, 130), (200, 640, 384), (1000, 384, 500), (2100, 130, 4100), (5000, 17, 2303), (4100, 272, 1000),
           (16384, 2048, 2048), (20000, 1000, 3001), (65536, 128, 1024), (33000, 60, 64), (33000, 512, 2048), (33333, 384, 66), (32768, 1152, 200),
           (45000, 776, 130)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,n", PRODUCT)
def test_product_of_whole_numbers(dev, rows, k, n, dt):
    """Products of at most 9, scaled by 2^0..3 by row and block and by 2^0..2 by block of the weight, sum to whole numbers below 2^24
    (9 * 32 * 4100, with bias and residual), and no eight of them spans 2^13: y is the exact result rounded once, in every form, and so
    is dx, for which y's operands change places."""
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(rows + k + n)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g, device=dev)
    each = lambda t, size, by: size.repeat_interleave(by, 1)[:, :t.shape[1]] * t
    x = each(ints(-3, 3, rows, k).double(), 2.0 ** ints(0, 3, rows, -(-k // 128)).double(), 128)
    w = ints(-3, 3, n, k).double()
    w = each(w, (2.0 ** ints(0, 2, -(-n // 128), -(-k // 128)).double()).repeat_interleave(128, 0)[:n], 128)
    bias, res, dy = ints(-9, 9, n), ints(-9, 9, rows, n), ints(-3, 3, rows, n)
    pw = ops.pack_weight_fp8(w.float(), transposed=True)
    want = x @ w.t()
    full = (want + bias + res).float().to(dt)                 # fp32 holds the sums: one rounding
    want = want.float().to(dt)
    x8 = ops.pack_fp8(x.to(dt))
    for a in (x.to(dt), x8, ops.pack_fp8(x.to(dt), "e5m2")):
        assert torch.equal(ops.linear_fp8(a, pw), want)
        y, _ = ops.linear_fp8(a, pw, bias=bias.float(), residual=res.to(dt), save=True)
        assert torch.equal(y, full)
    for fmt in ("e4m3", "e5m2"):
        dx, _, _ = ops.linear_fp8_backward(dy.to(dt), x8, pw, grad_fmt=fmt)
        assert torch.equal(dx, (dy.double() @ w).float().to(dt))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,c", [(1, 1), (9, 128), (7, 250), (33, 1001), (2, 2500), (16, 384)])
def test_packed_bytes(dev, rows, c, dt, fmt):
    """Every byte is the oracle's, padding included; only a NaN may be any of the type's NaNs, and a zero either zero."""
    from mad_amd import ops
    from oracle import fp8_ref as R
    g = torch.Generator().manual_seed(rows + c)
    x = (torch.randn((rows, c), generator=g) * torch.exp(4 * torch.randn((rows, c), generator=g))).to(dt)
    x[0, c // 3], x[rows - 1, c - 1] = float("nan"), -float("inf")
    q, s = R.stored(*R.pack_rows(x, fmt), fmt)
    p = ops.pack_fp8(x.to(dev), fmt)
    got = p.q.cpu().view(torch.uint8)
    nan = torch.isnan(q.view(R.TYPE[fmt]).float())
    assert torch.equal(torch.isnan(p.q.cpu().float()), nan)
    plain = lambda t: torch.where(t == 0x80, 0, t)[~nan]
    assert torch.equal(plain(got), plain(q)) and torch.equal(p.scale.cpu(), s)
    assert got.shape == (rows, (c + 15) // 16 * 16) and not bool(got[:, c:].any())


# the widest tensors there are on either side: rows, K, N
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,n", [(3, 1 << 20, 17), (70, (1 << 20) - 5, 24), (2, 40, 1 << 20), (70, 24, (1 << 20) - 3), (2048, 1 << 20, 2048)])
def test_widest_tensors(dev, rows, k, n, dt):
    """Whole numbers again: sums of 2^20 products of at most 9 stay below 2^24, so they are exact in any order (in the reference too)."""
    from mad_amd import ops
    g = torch.Generator(device=dev).manual_seed(k % 1000 + n % 1000)
    ints = lambda *s: torch.randint(-3, 4, s, generator=g, device=dev, dtype=torch.int8).to(torch.float32)
    x, w, dy = ints(rows, k), ints(n, k), ints(rows, n)
    pw = ops.pack_weight_fp8(w, transposed=True)
    want = (x @ w.t()).to(dt)
    y, x8 = ops.linear_fp8(x.to(dt), pw, save=True)
    assert torch.equal(y, want) and torch.equal(ops.linear_fp8(x.to(dt), pw), want)
    assert torch.equal(ops.unpack_fp8(x8).float(), x)
    dx, dw, db = ops.linear_fp8_backward(dy.to(dt), x8, pw)
    assert torch.equal(dx, (dy @ w).to(dt)) and torch.equal(dw, dy.t() @ x) and torch.equal(db, dy.sum(0))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_norm_of_the_widest_tensor(dev, dt):
    from mad_amd import ops
    c = 1 << 20
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((2, 1, 3, c), generator=g, device=dev).to(dt)
    coef = torch.randn((2, c, 2), generator=g, device=dev)
    y, p = ops.gn_apply_save(x, coef, act=True, drop_seed=9, drop_p=0.1)
    ref = ops.pack_fp8(x)
    assert torch.equal(y, ops.gn_apply(x, coef, act=True, drop_seed=9, drop_p=0.1))
    assert torch.equal(p.q.view(torch.uint8), ref.q.view(torch.uint8)) and torch.equal(p.scale, ref.scale)
    xr, yr = ops.gn_apply_restore(p, coef, act=True, drop_seed=9, drop_p=0.1)
    assert torch.equal(xr, ops.unpack_fp8(ref)) and torch.equal(yr, ops.gn_apply(xr, coef, act=True, drop_seed=9, drop_p=0.1))


@pytest.mark.parametrize("rows,k,n,dt", [(32768, 1152, 384, torch.bfloat16), (4100, 272, 1000, torch.bfloat16), (9000, 640, 521, torch.bfloat16),
                                         (5000, 777, 900, torch.float32), (31, 4096, 512, torch.float32)])
def test_large_forms_in_a_graph(dev, rows, k, n, dt):
    """Captured once and replayed on new inputs, with eager work between the replays: the eager results, bit for bit."""
    from mad_amd import ops

    def step(x, w, bias, dy):
        pw = ops.pack_weight_fp8(w, transposed=True)
        y, x8 = ops.linear_fp8(x, pw, bias=bias, save=True)
        return (y, ops.linear_fp8(x, pw, residual=y), *ops.linear_fp8_backward(dy, x8, pw))

    def inputs(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device=dev)
        return rand(rows, k).to(dt), rand(n, k) / math.sqrt(k), rand(n), rand(rows, n).to(dt)
    args = inputs(0)
    step(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*args)
    for seed in (1, 2, 3):
        fresh = inputs(seed)
        for t, v in zip(args, fresh):
            t.copy_(v)
        graph.replay()
        want = step(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
