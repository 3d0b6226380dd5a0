"""8-bit operators without a GPU: the oracle against torch's own 8-bit types, and every refusal before a launch."""
import ctypes

import pytest
import torch

torch.set_grad_enabled(False)


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_oracle_rounds_as_the_8_bit_type_does(fmt):
    from oracle import fp8_ref as R
    g = torch.Generator().manual_seed(1)
    top = R.MAX[fmt]
    u = torch.cat([torch.randn(4000, generator=g) * torch.exp(4 * torch.randn(4000, generator=g)),
                   torch.tensor([0.0, -0.0, top, -top, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -11, 2.0 ** -16, 2.0 ** -17, 3 * 2.0 ** -18,
                                 17.0, 19.0, 1.0625, 1.1875, float("nan")])])
    u = u[~(u.abs() > top)].float()
    want = u.to(R.TYPE[fmt]).double()
    assert torch.equal(torch.nan_to_num(R.round8(u.double(), fmt), 7.0), torch.nan_to_num(want, 7.0))


@pytest.mark.parametrize("fmt,top", [("e4m3", 448.0), ("e5m2", 57344.0)])
def test_oracle_exponent_is_the_smallest_that_fits(fmt, top):
    from oracle import fp8_ref as R
    for amax in (1.0, top, top * 1.0000001, top * 2, 1e-30, 3e38, 1e-45, 447.9, 1.75, 1.7500001):
        a = float(torch.tensor(amax, dtype=torch.float32))
        e = R.exponent(torch.tensor([a, -a / 3], dtype=torch.float64), fmt)
        assert a <= top * 2.0 ** e and (e == -126 or a > top * 2.0 ** (e - 1))
    assert R.exponent(torch.zeros(5), fmt) == 0
    assert R.exponent(torch.tensor([float("inf"), float("nan")]), fmt) == 0
    assert R.exponent(torch.tensor([float("inf"), 1.0]), fmt) == R.exponent(torch.tensor([1.0]), fmt)


# ------------------------------------------------------------------ refusals of the Python entry points
def _w(n, k, transposed=False):
    from mad_amd import ops
    e = lambda r, c: torch.zeros((r, (c + 15) // 16 * 16), dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = lambda r, c: torch.full((-(-r // 128), (-(-c // 128) + 3) // 4 * 4), 127, dtype=torch.uint8)
    return ops.Fp8Weight(e(n, k), s(n, k), (n, k), e(k, n) if transposed else None, s(k, n) if transposed else None)


def test_cpu_tensors_are_refused():
    from mad_amd import ops
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.pack_fp8(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.pack_weight_fp8(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.linear_fp8(x, _w(8, 32))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gn_apply_save(torch.zeros(1, 2, 2, 8), torch.zeros(1, 8, 2), act=True)
    p = ops.Fp8Tensor(torch.zeros((4, 32), dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros((4, 4), dtype=torch.uint8), (4, 32),
                      torch.float32)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.unpack_fp8(p)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gn_apply_restore(p._replace(shape=(1, 2, 2, 32)), torch.zeros(1, 32, 2), act=True)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.linear_fp8_backward(torch.zeros(4, 8), p, _w(8, 32, True))


def test_weights_that_do_not_fit_are_refused():
    from mad_amd import ops
    w = _w(8, 40)
    with pytest.raises(ValueError, match="do not belong"):
        ops.linear_fp8(torch.zeros(4, 40), w._replace(shape=(8, 50)))
    with pytest.raises(ValueError, match="do not belong"):
        ops.linear_fp8(torch.zeros(4, 40), w._replace(scale=w.scale[:, :2]))
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.linear_fp8(torch.zeros(4, 40), w._replace(q=w.q.view(torch.float8_e5m2)))


def test_trainer_options_are_checked():
    from mad_amd.train import UNetTrainer
    with pytest.raises(ValueError, match="checkpoints"):
        UNetTrainer(None, checkpoints="fp4")
    with pytest.raises(ValueError, match="products"):
        UNetTrainer(None, products="int8")


# ------------------------------------------------------------------ refusals of the C entry points (nothing is launched)
def _lib():
    from mad_amd import _lib
    return _lib.lib, _lib


P, ODD = 1 << 20, (1 << 20) + 8          # never read: every call below is refused on the host


def _refused(status, text):
    from mad_amd import _lib
    assert status != 0
    assert text in _lib.lib.mad_last_error().decode()


def test_c_pack_refusals():
    lib, L = _lib()
    ok = dict(rows=4, c=32)
    call = lambda x=P, dt=L.MAD_F32, fmt=L.MAD_E4M3, rows=4, c=32, q=P, s=P: lib.mad_pack_fp8(x, dt, fmt, rows, c, q, s, None)
    _refused(call(dt=7), "dtype")
    _refused(call(fmt=L.MAD_F32), "8-bit type")
    _refused(call(rows=-1), "bad shape")
    _refused(call(c=0), "bad shape")
    _refused(call(c=L.FP8_MAX_WIDTH + 1), "bad shape")
    _refused(call(x=None), "null")
    _refused(call(q=ODD), "aligned")
    _refused(call(s=P + 1), "aligned")
    assert call(x=None, q=None, s=None, rows=0) == 0
    call = lambda q=P, s=P, fmt=L.MAD_E4M3, rows=4, c=32, x=P, dt=L.MAD_F32: lib.mad_unpack_fp8(q, s, fmt, rows, c, x, dt, None)
    _refused(call(dt=2), "dtype")
    _refused(call(fmt=0), "8-bit type")
    _refused(call(c=-3), "bad shape")
    _refused(call(x=None), "null")
    _refused(call(q=ODD), "aligned")
    assert call(rows=0) == 0
    call = lambda w=P, dt=L.MAD_F32, n=8, k=8, q=P, s=P, qt=P, st=P: lib.mad_pack_weight_fp8(w, dt, n, k, q, s, qt, st, None)
    _refused(call(dt=3), "dtype")
    _refused(call(n=0), "bad shape")
    _refused(call(k=L.FP8_MAX_WIDTH + 1), "bad shape")
    _refused(call(st=None), "null")
    _refused(call(qt=ODD), "aligned")


@pytest.mark.parametrize("name", ["mad_gn_apply_save_fp8", "mad_gn_apply_restore_fp8"])
def test_c_norm_refusals(name):
    lib, L = _lib()
    fn = getattr(lib, name)
    save = "save" in name

    def call(x=P, coef=P, y=P, q=P, s=P, dt=L.MAD_BF16, B=1, HW=4, C=32, p=0.0):
        ptrs = (x, coef, y, q, s) if save else (q, s, coef, x, y)
        return fn(*ptrs, dt, B, HW, C, 1, 0, p, None)
    _refused(call(dt=2), "dtype")
    _refused(call(C=12), "multiple of 8")
    _refused(call(C=0), "multiple of 8")
    _refused(call(dt=L.MAD_F32, C=6), "multiple of 4")
    _refused(call(B=70000), "bad shape")
    _refused(call(HW=-1), "bad shape")
    _refused(call(p=1.0), "out of [0,1)")
    _refused(call(coef=None), "null")
    _refused(call(q=ODD), "aligned")
    _refused(call(y=ODD), "aligned")
    _refused(call(x=P + 2), "aligned")
    assert call(B=0) == 0 and call(HW=0) == 0


def test_c_linear_refusals():
    lib, L = _lib()

    def call(x=P, xt=L.MAD_E4M3, xs=P, w=P, ws=P, bias=None, res=None, y=P, dt=L.MAD_BF16, rows=4, K=32, N=8):
        return lib.mad_linear_fp8(x, xt, xs, w, ws, bias, res, y, dt, rows, K, N, None)
    _refused(call(dt=5), "dtype")
    _refused(call(xt=L.MAD_F32), "x is of type")
    _refused(call(rows=-2), "bad shape")
    _refused(call(K=0), "bad shape")
    _refused(call(N=L.FP8_MAX_WIDTH + 1), "bad shape")
    _refused(call(xs=None), "null")
    _refused(call(w=None), "null")
    _refused(call(w=ODD), "aligned")
    _refused(call(x=ODD), "aligned")
    _refused(call(rows=1 << 40, N=1 << 20), "need more")
    assert call(rows=0) == 0


def test_c_linear_save_refusals():
    lib, L = _lib()

    def call(x=P, dt=L.MAD_BF16, fmt=L.MAD_E4M3, w=P, ws=P, y=P, q=P, s=P, rows=1 << 20, K=32, N=8):
        return lib.mad_linear_fp8_save(x, dt, fmt, w, ws, None, None, y, q, s, rows, K, N, None)
    _refused(call(dt=5), "dtype")
    _refused(call(fmt=L.MAD_BF16), "8-bit type")
    _refused(call(rows=-1), "bad shape")
    _refused(call(N=0), "bad shape")
    _refused(call(K=0), "bad shape")
    _refused(call(w=None), "null")
    _refused(call(q=None), "null")
    _refused(call(q=ODD), "aligned")
    _refused(call(w=ODD), "aligned")
    _refused(call(rows=4, q=None), "null")
    assert call(rows=0) == 0
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_BF16, 8, 4096, 4096) == 0
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_BF16, 4096, 4096, 4096) == 1
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_BF16, 1 << 20, 256, 256) == 0
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_F32, 1 << 20, 256, 256) == 1


def test_c_wgrad_refusals():
    lib, L = _lib()

    def call(dy=P, dt=L.MAD_BF16, x=P, xt=L.MAD_E4M3, xs=P, dw=P, db=None, ws=P, nb=1 << 40, rows=4, N=8, K=32):
        return lib.mad_linear_fp8_wgrad(dy, dt, x, xt, xs, dw, db, ws, nb, rows, N, K, 0, 0, None)
    _refused(call(dt=2), "dtype")
    _refused(call(xt=L.MAD_BF16), "8-bit")
    _refused(call(N=0), "bad shape")
    _refused(call(rows=-1), "bad shape")
    _refused(call(dw=None), "null")
    _refused(call(x=ODD), "aligned")
    need = lib.mad_linear_fp8_wgrad_workspace(100000, 64, 64)
    assert need > 0
    _refused(call(rows=100000, N=64, K=64, nb=need - 1), "workspace")
    _refused(call(rows=100000, N=64, K=64, ws=None), "workspace")
    assert lib.mad_linear_fp8_wgrad_workspace(10, 64, 64) == 0
    assert lib.mad_linear_fp8_wgrad_workspace(-1, 64, 64) == 0


def test_types_agree_with_the_header():
    import os
    import re
    from mad_amd import _lib
    h = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mad_hip.h")).read()
    for name, v in (("MAD_E4M3", _lib.MAD_E4M3), ("MAD_E5M2", _lib.MAD_E5M2)):
        assert int(re.search(rf"#define {name} (\d+)", h).group(1)) == v
    a, b = re.search(r"#define MAD_FP8_MAX_WIDTH \((\d+) << (\d+)\)", h).groups()
    assert int(a) << int(b) == _lib.FP8_MAX_WIDTH
    assert ctypes.sizeof(ctypes.c_long) == 8


# ------------------------------------------------------------------ sizes that an int does not hold
@pytest.mark.parametrize("shape", [(1, 1 << 16, 1 << 16, 8), (1, 1 << 16, 1 << 15, 8), (1, (1 << 16) + 1, 1 << 16, 8), (65536, 1, 1, 8)])
def test_norm_refuses_sizes_beyond_the_entry_point(shape, monkeypatch):
    """H * W of 2^32 arrived at the C entry point as 0: it reported success and wrote nothing."""
    from mad_amd import _lib, ops
    monkeypatch.setattr(ops, "_fp8_dev", lambda *t: 0)
    monkeypatch.setattr(ops, "_fp8_call", lambda *a: pytest.fail("called"))
    empty = lambda s, dt: torch.empty(s, dtype=dt, device="meta")
    coef, rows = empty((shape[0], 8, 2), torch.float32), shape[0] * shape[1] * shape[2]
    with pytest.raises(ValueError, match="at most 65535 images"):
        ops.gn_apply_save(empty(shape, torch.bfloat16), coef, act=True)
    p = ops.Fp8Tensor(empty((rows, 16), torch.float8_e4m3fn), empty((rows, 4), torch.uint8), shape, torch.bfloat16)
    with pytest.raises(ValueError, match="at most 65535 images"):
        ops.gn_apply_restore(p, coef, act=True)


# ------------------------------------------------------------------ the built kernels
def _kernels():
    """Name -> metadata of every kernel in the built library (the notes of its gfx950 code objects)."""
    import struct
    from mad_amd import _lib
    msgpack = pytest.importorskip("msgpack")
    blob, magic, out = open(_lib.LIB_PATH, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", {}
    at = blob.find(magic)
    while at >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", blob, at + 24)[0]):
            offset, size, n = struct.unpack_from("<QQQ", blob, entry)
            target, entry = blob[entry + 24:entry + 24 + n], entry + 24 + n
            if b"gfx" not in target:
                continue
            elf = blob[at + offset:at + offset + size]
            table, (step, count) = struct.unpack_from("<Q", elf, 0x28)[0], struct.unpack_from("<HH", elf, 0x3a)
            for h in range(table, table + step * count, step):
                if struct.unpack_from("<I", elf, h + 4)[0] != 7:                 # SHT_NOTE
                    continue
                note = struct.unpack_from("<Q", elf, h + 0x18)[0]
                name, desc, _ = struct.unpack_from("<III", elf, note)
                start = note + 12 + ((name + 3) & ~3)
                for k in msgpack.unpackb(elf[start:start + desc])["amdhsa.kernels"]:
                    out[k[".name"]] = k
        at = blob.find(magic, at + 24)
    return out


def test_kernels_keep_their_registers():
    """None of them spills: a reload from scratch memory waits for every copy in flight."""
    found = {n: k[".private_segment_fixed_size"] for n, k in _kernels().items() if "fp8" in n}
    assert len(found) > 50
    assert not {n: v for n, v in found.items() if v}


def test_launches_stay_below_the_threads_they_count():
    """A launch counts fewer than 2^32 threads: longer inputs are packed first, or refused."""
    lib, L = _lib()
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_BF16, (1 << 30) - 128, 8, 8) == 0
    assert lib.mad_linear_fp8_needs_pack(P, L.MAD_BF16, 1 << 30, 8, 8) == 1
    _refused(lib.mad_linear_fp8(P, L.MAD_BF16, None, P, P, None, None, P, L.MAD_BF16, 1 << 28, 5, 16, None), "need more")
    _refused(lib.mad_linear_fp8(P, L.MAD_F32, None, P, P, None, None, P, L.MAD_F32, 1 << 20, 8, 1 << 15, None), "need more")


def test_rounding_is_as_small_as_documented():
    """e4m3: at most 2^-4 of an element down to 2^-13 of its block's largest, at most 2^-17 of the largest below, zero from 2^-19 on."""
    from oracle import fp8_ref as R
    g = torch.Generator().manual_seed(2)
    for top in (1.0, 1.75, 1.7500002, 3.4e5, 2.0 ** -40):
        ratio = torch.cat([2.0 ** (-21 * torch.rand(126, generator=g)), torch.tensor([2.0 ** -19])])
        x = torch.cat([torch.tensor([top]), top * ratio]).float()
        v = R.pack_rows(x[None])[0][0]
        err, x = (v - x.double()).abs(), x.double()
        near, far = x >= x[0] * 2.0 ** -13, x <= x[0] * 2.0 ** -19
        assert bool((err <= torch.where(near, x * 2.0 ** -4, x[0] * 2.0 ** -17)).all()) and bool((v[far] == 0).all())
