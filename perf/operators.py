"""The 8-bit operators of the training and serving paths as measurable cases.

Two operators and the format they share:

* the matrix product of 8-bit operands with one power-of-two scale per block of 128 (``ops.linear_fp8``) with its
  gradients (``ops.linear_fp8_backward``), and the packing of weights (``ops.pack_weight_fp8``);
* activation checkpoints in 8 bits: ``ops.pack_fp8`` / ``ops.unpack_fp8``, and the passes that apply a GroupNorm while
  they store or restore its input (``ops.gn_apply_save`` / ``ops.gn_apply_restore``).

The format: a row is cut into blocks of 128 elements (the last one may be shorter).  A block's scale is 2^e with the
smallest integer e >= -126 for which its largest finite magnitude is at most MAX * 2^e (e4m3: MAX = 448, e5m2: 57344; a
block of zeros has e = 0); its elements are x * 2^-e rounded to nearest even.  Weights (N, K) have one scale per
128 x 128 block.  Stored rows are padded with zeros to whole 16 bytes, scales (one byte, e + 127) to whole groups of four.
"""
import math

import torch

own = False

BLOCK = 128
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # one image's timestep embedding through a 768 x 768 layer: a single row, where latency is all there is
        {"name": "token", "op": "linear", "rows": 1, "k": 768, "n": 768, "dtype": "bf16", "bias": True, "residual": False},
        # one decoding step of 32 sequences: the weights are read once and the rows hardly count
        {"name": "tokens_32", "op": "linear", "rows": 32, "k": 4096, "n": 8192, "dtype": "bf16", "bias": False, "residual": False},
        # fp32 parity mode at sizes that fill no tile and no block
        {"name": "ragged", "op": "linear", "rows": 777, "k": 1000, "n": 328, "dtype": "fp32", "bias": True, "residual": False},
        # qkv projection of the 32 x 32 attention blocks of the 256 x 256 model, batch 32
        {"name": "qkv_256", "op": "linear", "rows": 32768, "k": 256, "n": 768, "dtype": "bf16", "bias": True, "residual": False},
        # output projection with its residual, 32 x 32 blocks of the 64 x 64 model, batch 64
        {"name": "proj_64", "op": "linear", "rows": 65536, "k": 384, "n": 384, "dtype": "bf16", "bias": True, "residual": True},
        # a wide layer over a long batch: bound by the matrix units
        {"name": "wide", "op": "linear", "rows": 16384, "k": 4096, "n": 8192, "dtype": "bf16", "bias": False, "residual": False},
        # one training pass of a small layer in fp32, sizes that fill no tile
        {"name": "train_ragged", "op": "train", "rows": 501, "k": 200, "n": 137, "dtype": "fp32", "grad": "e4m3"},
        # one training pass of the 64 x 64 model's qkv projection, batch 64
        {"name": "train_qkv", "op": "train", "rows": 65536, "k": 384, "n": 1152, "dtype": "bf16", "grad": "e4m3"},
        # one training pass of a wide layer, gradients in the type with the wider range
        {"name": "train_wide", "op": "train", "rows": 8192, "k": 4096, "n": 4096, "dtype": "bf16", "grad": "e5m2"},
        # a checkpoint of the 8 x 8 stage at batch 2: latency
        {"name": "save_8x8", "op": "norm", "b": 2, "h": 8, "w": 8, "c": 512, "dtype": "bf16", "act": True},
        # a checkpoint of the 128 x 128 stage of the 256 x 256 model at batch 32: bandwidth
        {"name": "save_128x128", "op": "norm", "b": 32, "h": 128, "w": 128, "c": 256, "dtype": "bf16", "act": True},
        # an fp32 tensor of odd width packed and restored
        {"name": "pack_odd", "op": "pack", "rows": 4099, "k": 1001, "dtype": "fp32", "fmt": "e4m3"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "train", "train", "norm", "pack"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    if op in ("linear", "train"):
        most = 1.0e12 if op == "linear" else 0.8e12
        # widths in whole sixteens twice out of three times, any width otherwise
        g = rng.choice((16, 16, 1))
        k, n = (max(1, _log(rng, 32, 6144) // g) * g for _ in range(2))
        per_row = (2.0 if op == "linear" else 6.0) * k * n
        per_row_bytes = BYTES[dtype] * (k + 2 * n if op == "linear" else 2 * k + 2 * n)
        rows = _log(rng, 1, max(1, min(65536, int(most / per_row), int(1.2e9 / per_row_bytes))))
        if op == "train":
            return {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "grad": rng.choice(("e4m3", "e4m3", "e5m2"))}
        return {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.6, "residual": rng.random() < 0.3}
    if op == "norm":
        c = 8 * _log(rng, 4, 128)
        side = _log(rng, 4, 128)
        other = _log(rng, 4, 128)
        b = _log(rng, 1, max(1, min(32, (1 << 26) // (side * other * c))))
        return {"op": op, "b": b, "h": side, "w": other, "c": c, "dtype": dtype, "act": rng.random() < 0.7}
    k = _log(rng, 1, 5000)
    return {"op": op, "rows": _log(rng, 1, min(200000, (1 << 26) // k)), "k": k, "dtype": dtype, "fmt": rng.choice(("e4m3", "e5m2"))}


# ---------------------------------------------------------------------------------------------- inputs
def _up(n, m):
    return -(-n // m) * m


def _two(e):
    """2^e of whole numbers -126..127, exactly (a power function may be off by an ulp)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _weight(w):
    """(q, scale) of a weight in the stored format: what a program that serves the layer loads from its checkpoint."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    full = torch.zeros((nb * BLOCK, kb * BLOCK), device=w.device)
    full[:n, :k] = w
    tiles = full.view(nb, BLOCK, kb, BLOCK)
    m, e = torch.frexp(tiles.abs().amax((1, 3)))
    e = e - torch.where(m <= 0.875, 9, 8)
    q = torch.zeros((n, _up(k, 16)), device=w.device)
    q[:, :k] = (tiles * _two(-e)[:, None, :, None]).reshape(nb * BLOCK, kb * BLOCK)[:n, :k]
    scale = torch.full((nb, _up(kb, 4)), 127, dtype=torch.uint8, device=w.device)
    scale[:, :kb] = (e + 127).to(torch.uint8)
    return q.to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    dt = DTYPE[case["dtype"]]
    st = dict(case)
    if case["op"] == "norm":
        # a convolution's output before its GroupNorm: some channels are larger than others; the (a, d) pairs undo it
        b, h, w, c = (case[x] for x in "bhwc")
        size = torch.exp(0.5 * rand(c))
        st["x"] = (rand(b, h, w, c) * size + 0.3 * rand(c)).to(dt)
        a = (1.0 + 0.2 * rand(b, c)) / size
        st["coef"] = torch.stack((a, 0.2 * rand(b, c)), -1).contiguous()
        return st
    rows, k = case["rows"], case["k"]
    # activations after a norm: unit size with a spread between channels
    st["x"] = (rand(rows, k) * torch.exp(0.4 * rand(k))).to(dt)
    if case["op"] == "pack":
        return st
    n = case["n"]
    weight = rand(n, k) / math.sqrt(k)
    st["bias"] = 0.1 * rand(n) if case.get("bias") else None
    st["residual"] = rand(rows, n).to(dt) if case.get("residual") else None
    if case["op"] == "linear":
        st["q"], st["scale"] = _weight(weight)
    else:
        # a training pass holds the fp32 master weights; gradients differ in size from row to row
        st["weight"], st["bias"] = weight, 0.1 * rand(n)
        st["dy"] = (1e-3 * rand(rows, n) * torch.exp(rand(rows, 1))).to(dt)
    return st


# ---------------------------------------------------------------------------------------------- plain form
def _rounded(x, fmt):
    """The values that the rows of x (..., K) stand for after packing, in fp32."""
    k = x.shape[-1]
    kb = -(-k // BLOCK)
    t = torch.nn.functional.pad(x.float().reshape(-1, k), (0, kb * BLOCK - k)).view(-1, kb, BLOCK)
    m, e = torch.frexp(t.abs().amax(-1, keepdim=True))
    e = torch.where(m == 0, 0, e - torch.where(m <= 0.875, 9, 8) - (0 if fmt == "e4m3" else 7)).clamp_min(-126)
    v = (t * _two(-e)).to(FP8[fmt]).float() * _two(e)
    return v.view(-1, kb * BLOCK)[:, :k].reshape(x.shape)


def _rounded_weight(w):
    """The values a weight stands for after packing, in fp32."""
    q, scale = _weight(w)
    return _weight_values(q, scale, *w.shape)


def _weight_values(q, scale, n, k):
    size = _two(scale.int() - 127).repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return q[:, :k].float() * size


def _normed(x, coef, act):
    """act(x * a + d) in fp32, (a, d) per sample and channel."""
    t = x.float() * coef[:, None, None, :, 0] + coef[:, None, None, :, 1]
    return t / (1.0 + torch.exp(-t)) if act else t


def run(state):
    op, dt, x = state["op"], DTYPE[state["dtype"]], state["x"]
    if own:
        from mad_amd import ops
        if op == "linear":
            w = ops.Fp8Weight(state["q"], state["scale"], (state["n"], state["k"]))
            return ops.linear_fp8(x, w, bias=state["bias"], residual=state["residual"])
        if op == "train":
            w = ops.pack_weight_fp8(state["weight"], transposed=True)
            y, x8 = ops.linear_fp8(x, w, bias=state["bias"], save=True)
            dx, dw, db = ops.linear_fp8_backward(state["dy"], x8, w, grad_fmt=state["grad"])
            return y, dx, dw, db
        if op == "norm":
            h, x8 = ops.gn_apply_save(x, state["coef"], act=state["act"])
            xr, hr = ops.gn_apply_restore(x8, state["coef"], act=state["act"])
            return h, xr, hr
        return ops.unpack_fp8(ops.pack_fp8(x, fmt=state["fmt"]))
    if op == "linear":
        y = _rounded(x, "e4m3") @ _weight_values(state["q"], state["scale"], state["n"], state["k"]).t()
        if state["bias"] is not None:
            y = y + state["bias"]
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(dt)
    if op == "train":
        xr, w, dy = _rounded(x, "e4m3"), _rounded_weight(state["weight"]), state["dy"].float()
        y = xr @ w.t() + state["bias"]
        return y.to(dt), (_rounded(state["dy"], state["grad"]) @ w).to(dt), dy.t() @ xr, dy.sum(0)
    if op == "norm":
        xr = _rounded(x, "e4m3").to(dt)
        return _normed(x, state["coef"], state["act"]).to(dt), xr, _normed(xr, state["coef"], state["act"]).to(dt)
    return _rounded(x, state["fmt"]).to(dt)


def work(case):
    s = BYTES[case["dtype"]]
    if case["op"] == "norm":
        # x in, h out, the checkpoint out; the checkpoint in, x and h out; (a, d) each time
        n, pixels = case["b"] * case["h"] * case["w"] * case["c"], case["b"] * case["h"] * case["w"]
        packed = n + pixels * -(-case["c"] // BLOCK)
        return {"bytes": 4 * s * n + 2 * packed + 2 * 8 * case["b"] * case["c"], "flops": (14 if case["act"] else 6) * n}
    rows, k = case["rows"], case["k"]
    packed = rows * k + rows * -(-k // BLOCK)
    if case["op"] == "pack":
        return {"bytes": 2 * s * rows * k + 2 * packed, "flops": 3 * rows * k}
    n = case["n"]
    if case["op"] == "linear":
        b = s * rows * (k + n) + n * k + (4 * n if case["bias"] else 0) + (s * rows * n if case["residual"] else 0)
        return {"bytes": b, "flops": 2 * rows * k * n}
    # x, dy, the weights and the bias in; y, dx and the fp32 gradients out; the checkpoint out and in
    return {"bytes": s * rows * (2 * k + 2 * n) + 2 * packed + 8 * n * k + 8 * n, "flops": 6 * rows * k * n}


# ---------------------------------------------------------------------------------------------- 64 bits
def _pow2(e):
    """2^e in fp64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _near(x, fmt, dims):
    """x (fp64) rounded to 8 bits over blocks whose largest magnitude is taken over `dims`: from the definition."""
    digits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    top = x.abs().amax(dims, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, TOP[fmt]) / TOP[fmt]))
    e = torch.where(top > TOP[fmt] * _pow2(e), e + 1, e)
    e = torch.where((top <= TOP[fmt] * _pow2(e - 1)) & (top > 0), e - 1, e).clamp_min(-126)
    u = x / _pow2(e)
    mag = torch.floor(torch.log2(u.abs().clamp_min(2.0 ** (low - digits - 2))))
    mag = torch.where(_pow2(mag + 1) <= u.abs(), mag + 1, mag)
    mag = torch.where(_pow2(mag) > u.abs(), mag - 1, mag)
    step = _pow2(mag.clamp_min(low) - digits)
    return torch.round(u / step) * step * _pow2(e)


def _near_rows(x, fmt="e4m3"):
    x = x.double()
    k = x.shape[-1]
    whole = k // BLOCK * BLOCK
    parts = []
    if whole:
        parts.append(_near(x[..., :whole].unflatten(-1, (-1, BLOCK)), fmt, -1).flatten(-2))
    if whole < k:
        parts.append(_near(x[..., whole:], fmt, -1))
    return torch.cat(parts, -1)


def _near_weight(w):
    n, k = w.shape
    whole = torch.nn.functional.pad(w.double(), (0, -k % BLOCK, 0, -n % BLOCK))
    tiles = whole.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))
    return _near(tiles, "e4m3", (1, 3)).flatten(2).flatten(0, 1)[:n, :k]


def _stored_weight(q, scale, n, k):
    size = _pow2(scale.long() - 127)
    r, c = torch.arange(n, device=q.device) // BLOCK, torch.arange(k, device=q.device) // BLOCK
    return q[:, :k].double() * size[r][:, c]


def _act64(x, coef, act):
    coef = coef.double()
    t = x * coef[:, None, None, :, 0] + coef[:, None, None, :, 1]
    return t * torch.sigmoid(t) if act else t


def exact(case, seed):
    st = prepare(case, seed)
    op, x = case["op"], st["x"]
    if op == "linear":
        y = _near_rows(x) @ _stored_weight(st["q"], st["scale"], case["n"], case["k"]).t()
        if st["bias"] is not None:
            y += st["bias"].double()
        if st["residual"] is not None:
            y += st["residual"].double()
        return y
    if op == "train":
        xr, w, dy = _near_rows(x), _near_weight(st["weight"]), st["dy"].double()
        return xr @ w.t() + st["bias"].double(), _near_rows(dy, case["grad"]) @ w, dy.t() @ xr, dy.sum(0)
    if op == "norm":
        xr = _near_rows(x)
        return _act64(x.double(), st["coef"], case["act"]), xr, _act64(xr, st["coef"], case["act"])
    return _near_rows(x, case["fmt"])
