"""layer_norm, dropout and dropout_add_layer_norm (lbm_amd/training.py) against the float64 / integer oracle.

Error bounds.  u(T) = finfo(T).eps / 2 is one rounding to T, e = 2^-24 one to fp32.  A row's sums are made of at most
depth(D) = 8 ceil(D / 2048) + 32 dependent fp32 additions (eight a chunk in a thread, a tree over lanes and waves), so a mean is off by
(depth + 2) e mean|z|, and
  E = e (depth + 16) rstd (mean|z| + |z| + |x scale|) + e (depth + 16) 2 |xhat|      bounds the error of xhat
(the first part: mean and the join's own roundings; the second: the variance's sum, square root, division, product).  From there
  y      u |y| + |w| E + 4 e (|xhat w| + |b|)
  dz     u |dz| + rstd (4 e |g| + e (depth + 4) mean|g| + |xhat| (e (depth + 4) mean|g xhat| + mean(|g| E)) + E |mean(g xhat)|) + e (depth + 16) |dz|
  dx     that times scale, its own rounding, and 4 e |dx|
  dw     u |dw| + sum |dy| E + e n sum |dy xhat|     n = rows summed in sequence, at most rows / 64 + 64 (fewer rows: all), + 32
  db     u |db| + e n sum |dy|
and half of the smallest subnormal of f16 where results are that small.
"""
import ctypes as C
import math

import pytest
import torch

from lbm_amd import dropout, dropout_add_layer_norm, hip, layer_norm
from oracle import train_ref as ref

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E32 = 2.0 ** -24
gpu = pytest.mark.gpu


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == F16 else 0.0


def bounds(o, eps, dtype_y, dtype_x, dtype_p, scale=1.0):
    """Tolerances of y, dresidual / dz, dx, dweight, dbias (docstring above)."""
    D = o["z"].shape[-1]
    rows = o["z"].numel() // D
    depth = 8 * math.ceil(D / 2048) + 32
    mean = lambda t: t.mean(-1, keepdim=True)        # noqa: E731
    E = E32 * (depth + 16) * (o["rstd"] * (mean(o["z"].abs()) + o["z"].abs() + o["xs"].abs()) + 2 * o["xhat"].abs())
    t = {"y": u(dtype_y) * o["y"].abs() + o["w"].abs() * E + 4 * E32 * ((o["xhat"] * o["w"]).abs() + o["b"].abs()) + tiny(dtype_y)}
    if "dy" in o:
        g, xh, dz = o["g"].abs(), o["xhat"].abs(), o["dresidual"].abs()
        raw = o["rstd"] * (4 * E32 * g + E32 * (depth + 4) * mean(g) + xh * (E32 * (depth + 4) * mean(g * xh) + mean(g * E)) + E * o["c2"].abs()) \
            + E32 * (depth + 16) * dz
        t["dresidual"] = u(dtype_y) * dz + raw + tiny(dtype_y)
        t["dx"] = u(dtype_x) * o["dx"].abs() + raw * scale + 4 * E32 * o["dx"].abs() + tiny(dtype_x)
        n = min(rows, rows / 64 + 64) + 32
        flat = lambda v: v.reshape(-1, D).sum(0)     # noqa: E731
        t["dweight"] = u(dtype_p) * o["dweight"].abs() + flat(o["dy"].abs() * E) + E32 * n * flat((o["dy"] * o["xhat"]).abs()) + tiny(dtype_p)
        t["dbias"] = u(dtype_p) * o["dbias"].abs() + E32 * n * flat(o["dy"].abs()) + tiny(dtype_p)
    return t


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.2f} of the bound"


def operands(shape, x_type, res_type, p_type, affine, seed, offset_rows=0.3):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    x = torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g)) + offset_rows * torch.randn(*shape[:-1], 1, generator=g)
    r = torch.randn(*shape, generator=g)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    b = 0.2 * torch.randn(D, generator=g)
    dy = torch.randn(*shape, generator=g)
    out = dict(x=x.to(x_type), residual=None if res_type is None else r.to(res_type), weight=w.to(p_type) if affine in ("both", "weight") else None,
               bias=b.to(p_type) if affine in ("both", "bias") else None, dy=dy.to(res_type or x_type))
    return {k: None if v is None else v.cuda() for k, v in out.items()}


def check(o, p=0.0, seed=0, offset=0, eps=1e-5, x_view=None):
    """Forward without gradients, then forward and backward, of the operator that the operands ask for."""
    joined = o["residual"] is not None
    x = o["x"] if x_view is None else x_view
    D = x.shape[-1]
    factor = None
    if joined and p > 0:
        factor = ref.keep(tuple(x.shape), p, seed, offset).double() * ref.scale(p)
    want = ref.norm(x, o["weight"], o["bias"], eps, o["residual"], factor, o["dy"])
    given = [o[k] for k in ("weight", "bias") if o[k] is not None]
    tol = bounds(want, eps, o["dy"].dtype, x.dtype, given[0].dtype if given else x.dtype, ref.scale(p) if joined else 1.0)

    def call(x, residual, weight, bias):
        if joined:
            return dropout_add_layer_norm(x, residual, weight, bias, p=p, seed=seed, offset=offset, eps=eps)
        return layer_norm(x, weight, bias, eps)

    plain = call(x, o["residual"], o["weight"], o["bias"])
    assert plain.dtype == o["dy"].dtype and plain.is_contiguous() and not plain.requires_grad
    within(plain, want["y"], tol["y"], "y")
    leaves = {k: (x if k == "x" else o[k]).detach().requires_grad_() for k in ("x", "residual", "weight", "bias") if k == "x" or o[k] is not None}
    y = call(leaves["x"], leaves.get("residual"), leaves.get("weight"), leaves.get("bias"))
    assert torch.equal(y.detach().view(torch.uint8) if y.numel() else y, plain.view(torch.uint8) if y.numel() else plain)     # with and without statistics: the same bits
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), o["dy"])))
    for k, t in grads.items():
        assert t.dtype == leaves[k].dtype
        within(t, want["d" + k], tol["d" + k], "d" + k)
    return want, grads


# ---------------------------------------------------------------------------------------------- CPU: the oracle, refusals

def test_oracle_generator_known_answers():
    """The published test vectors of Philox4x32-10."""
    f = 0xFFFFFFFF
    for ctr, key, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ((f, f, f, f), (f, f), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in ref.philox4x32(ctr, key)) == want


def test_oracle_mask_rate():
    """Kept elements of 2^20: the count is binomial; 6 standard deviations."""
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        k = int(ref.keep((n,), p, 1234, 5).sum())
        assert abs(k - n * (1 - p)) < 6 * math.sqrt(n * p * (1 - p))
    assert not torch.equal(ref.keep((n,), 0.5, 1234, 5), ref.keep((n,), 0.5, 1234, 6))


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    D = 7
    t = {k: torch.randn(*s, generator=g, dtype=torch.float64) for k, s in (("x", (3, D)), ("r", (3, D)), ("w", (D,)), ("b", (D,)), ("dy", (3, D)))}
    factor = ref.keep((3, D), 0.3, 9, 2).double() * ref.scale(0.3)
    o = ref.norm(t["x"], t["w"], t["b"], 1e-5, t["r"], factor, t["dy"])
    loss = lambda: (ref.norm(t["x"], t["w"], t["b"], 1e-5, t["r"], factor)["y"] * t["dy"]).sum()     # noqa: E731
    for k, name in (("x", "dx"), ("r", "dresidual"), ("w", "dweight"), ("b", "dbias")):
        v = torch.randn(t[k].shape, generator=g, dtype=torch.float64)
        keep, h = t[k].clone(), 1e-5
        t[k] = keep + h * v
        up = loss()
        t[k] = keep - h * v
        down = loss()
        t[k] = keep
        assert abs(float((up - down) / (2 * h) - (o[name] * v).sum())) < 1e-8        # h^2 third derivatives (~100) and 1e-16 / h


def _desc(**kw):
    a = torch.zeros(64)
    d = hip.NormDesc()
    d.x = d.y = d.dy = d.dx = a.data_ptr()
    d.mean = d.rstd = a.data_ptr()
    d.rows, d.cols, d.ld_x, d.ld_residual, d.ld_dy, d.eps = 2, 8, 8, 8, 8, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d, a


@pytest.mark.parametrize("kw,message", [
    (dict(cols=0), b"bad sizes"), (dict(rows=-1), b"bad sizes"), (dict(cols=(1 << 28) + 1, ld_x=1 << 29), b"bad sizes"),
    (dict(x_type=3), b"element type"), (dict(param_type=-1), b"element type"), (dict(res_type=1), b"res_type"),
    (dict(x_type=1, res_type=0), b"res_type"), (dict(x_type=1, res_type=1, param_type=2), b"param_type"), (dict(ld_x=7), b"row stride"),
    (dict(eps=0.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(x=None), b"null x"),
    (dict(p=0.5), b"residual"), (dict(p=float("nan")), b"residual"), (dict(x=2), b"aligned")])
def test_abi_refusals_of_both_passes(kw, message):
    lib = hip.load()
    d, _keep = _desc(**kw)
    for fn in (lib.lbm_hip_norm_forward, lib.lbm_hip_norm_backward):
        assert fn(C.byref(d), None) != 0
        assert message in lib.lbm_hip_last_error(), lib.lbm_hip_last_error()


def test_abi_refusals_of_one_pass():
    lib = hip.load()
    assert lib.lbm_hip_norm_forward(None, None) != 0 and b"null descriptor" in lib.lbm_hip_last_error()
    for kw, msg in ((dict(y=None), b"null y"), (dict(mean=None), b"go together"), (dict(residual=64, p=1.5), b"not a probability"),
                    (dict(residual=64, ld_residual=4), b"row stride"), (dict(seed_dev=4), b"seed")):
        d, _keep = _desc(**kw)
        assert lib.lbm_hip_norm_forward(C.byref(d), None) != 0 and msg in lib.lbm_hip_last_error(), (kw, lib.lbm_hip_last_error())
    for kw, msg in ((dict(dy=None), b"null dy"), (dict(rstd=None), b"null dy"), (dict(ld_dy=1), b"row stride"), (dict(dresidual=64), b"without a residual"),
                    (dict(dweight=64), b"workspace"), (dict(dbias=64, workspace=64, workspace_bytes=8), b"workspace"),
                    (dict(dbias=64, workspace=68, workspace_bytes=1 << 40), b"workspace")):
        d, _keep = _desc(**kw)
        assert lib.lbm_hip_norm_backward(C.byref(d), None) != 0 and msg in lib.lbm_hip_last_error(), (kw, lib.lbm_hip_last_error())
    a = torch.zeros(64)
    for args, msg in (((a.data_ptr(), a.data_ptr(), -1, 0, 0.5, 1, None, 0), b"bad size"), ((a.data_ptr(), a.data_ptr(), 8, 7, 0.5, 1, None, 0), b"element type"),
                      ((a.data_ptr(), a.data_ptr(), 8, 0, -0.1, 1, None, 0), b"probability"), ((a.data_ptr(), a.data_ptr(), 8, 0, float("nan"), 1, None, 0), b"probability"),
                      ((None, a.data_ptr(), 8, 0, 0.5, 1, None, 0), b"null"), ((a.data_ptr() + 2, a.data_ptr(), 8, 0, 0.5, 1, None, 0), b"aligned")):
        assert lib.lbm_hip_dropout(*args, None) != 0 and msg in lib.lbm_hip_last_error(), lib.lbm_hip_last_error()
    for bad in ((-1, 8), (1, 0), (1 << 45, 1 << 10), (1, (1 << 28) + 1)):
        assert lib.lbm_hip_norm_workspace_bytes(*bad) == 0
    assert lib.lbm_hip_norm_workspace_bytes(0, 8) > 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    for call in (lambda: layer_norm(x), lambda: dropout(x, 0.5, 1), lambda: dropout_add_layer_norm(x, x)):
        with pytest.raises(hip.HipError, match="GPU"):
            call()


# ---------------------------------------------------------------------------------------------- dropout

SIZES = [1, 7, 8, 9, 511, 2048, 2049, 100003]


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", SIZES)
def test_dropout_bits(dtype, n):
    """The mask and the values, bit for bit: one fp32 product, one rounding."""
    for k, p in enumerate((0.1, 0.5, 1 / 3, 0.999)):
        x = torch.randn(n, generator=torch.Generator().manual_seed(n + k)).to(dtype)
        seed, offset = 0x9E3779B97F4A7C15 * (k + 1) % 2 ** 64, 2 ** 63 + k
        m = ref.keep((n,), p, seed, offset)
        want = torch.where(m, x.float() * torch.tensor(ref.scale(p), dtype=F32), torch.zeros(())).to(dtype)
        leaf = x.cuda().requires_grad_()
        y = dropout(leaf, p, seed, offset)
        assert torch.equal(y.detach().cpu(), want)
        assert torch.equal(dropout(leaf.detach(), p, seed, offset).cpu(), want)
        dy = torch.randn(n, generator=torch.Generator().manual_seed(n + k + 99)).to(dtype)
        dx, = torch.autograd.grad(y, leaf, dy.cuda())
        assert torch.equal(dx.cpu(), torch.where(m, dy.float() * torch.tensor(ref.scale(p), dtype=F32), torch.zeros(())).to(dtype))


@gpu
def test_dropout_border_of_the_threshold():
    """p chosen so that the threshold is an element's own number (kept) and one above it (dropped): the lower 16 bits decide."""
    n, seed, offset = 4096, 77, 3
    r = ref.numbers(0, n, seed, offset)
    x = torch.ones(n, device="cuda")
    for e in (0, 1, 6, 7, 8, 1001, 4095):
        for up in (0, 1):
            p = (int(r[e]) + up) / 2 ** 32
            y = dropout(x, p, seed, offset).cpu()
            assert torch.equal(y != 0, ref.keep((n,), p, seed, offset))
            assert bool(y[e] != 0) == (up == 0)


@gpu
def test_dropout_extremes():
    x = torch.tensor([1.0, -2.0, float("inf"), float("-inf"), float("nan")] * 100, device="cuda")
    assert torch.equal(dropout(x, 0.0, 5).nan_to_num(7.0), x.nan_to_num(7.0))
    assert torch.equal(dropout(x, 2.0 ** -34, 5).nan_to_num(7.0), x.nan_to_num(7.0))       # rounds to zero
    for p in (1.0, 1 - 2.0 ** -34):
        assert torch.equal(dropout(x, p, 5), torch.zeros_like(x))                          # no inf * 0
    m = ref.keep((500,), 0.5, 5, 0).cuda()
    y = dropout(x, 0.5, 5)
    assert torch.equal(y[~m], torch.zeros_like(y[~m])) and torch.equal(y[m].nan_to_num(7.0), (2 * x[m]).nan_to_num(7.0))
    assert dropout(x[:0], 0.5, 5).shape == (0,)
    assert dropout(torch.ones((), device="cuda"), 0.5, 1).shape == ()


@gpu
def test_dropout_seeds_and_layouts():
    x = torch.randn(37, 19, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    want = dropout(x, 0.3, -5, 11)
    assert torch.equal(want, dropout(x, 0.3, 2 ** 64 - 5, 11))
    assert torch.equal(want, dropout(x, 0.3, torch.tensor([-5], device="cuda"), 11))
    assert torch.equal(want, dropout(x, 0.3, torch.tensor(-5, device="cuda"), 11))
    assert torch.equal(want, dropout(x.view(19, 37), 0.3, -5, 11).view(37, 19))            # the row-major index counts, not the shape
    assert torch.equal(want, dropout(x.t().contiguous().t(), 0.3, -5, 11))                 # nor the strides
    wide = torch.zeros(37, 40, device="cuda")
    wide[:, 3:22] = x
    assert torch.equal(want, dropout(wide[:, 3:22], 0.3, -5, 11))
    flat = torch.zeros(37 * 19 + 1, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.equal(want, dropout(flat[1:].view(37, 19), 0.3, -5, 11))                  # starts four bytes into an allocation
    half = torch.zeros(37 * 19 + 1, device="cuda", dtype=F16)
    half[1:] = x.reshape(-1)
    assert torch.equal(dropout(half[1:], 0.3, -5, 11), dropout(x.half().reshape(-1), 0.3, -5, 11))
    one = x[:1].expand(37, 19)
    assert torch.equal(dropout(one, 0.3, -5, 11), dropout(one.contiguous(), 0.3, -5, 11))
    for bad in (dict(p=1.5), dict(p=-0.1), dict(p=float("nan")), dict(seed=1 << 64), dict(seed=-(1 << 63) - 1), dict(offset=-1), dict(offset=1 << 64),
                dict(seed=torch.zeros(2, device="cuda", dtype=torch.int64)), dict(seed=torch.zeros(1, device="cuda")), dict(seed=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(hip.HipError):
            dropout(x, **{**dict(p=0.5, seed=1), **bad})
    with pytest.raises(TypeError):
        dropout(x, 0.5, 1.5)
    with pytest.raises(hip.HipError):
        dropout(x.double(), 0.5, 1)


@gpu
def test_dropout_beyond_32_bit_indexes():
    n = (1 << 32) + 4099
    x = torch.ones(n, device="cuda", dtype=F16)
    y = dropout(x, 0.25, 42, 7)
    del x
    for first in (0, (1 << 31) - 1000, (1 << 32) - 1000, n - 2000):
        assert torch.equal((y[first:first + 2000] != 0).cpu(), ref.keep((2000,), 0.25, 42, 7, first=first))


# ---------------------------------------------------------------------------------------------- layer_norm and the join

TYPES = [(F32, None, F32), (F16, None, F32), (BF16, None, BF16), (F32, F32, F32), (F16, F16, F16), (BF16, BF16, F32), (F16, F32, F32), (BF16, F32, BF16)]
SHAPES = [(1, 1), (5, 1), (3, 2), (1, 7), (4, 8), (130, 16), (67, 24), (33, 100), (9, 255), (700, 256), (41, 257), (19, 512), (13, 520), (7, 1021), (6, 1024),
          (5, 1537), (4, 2048), (3, 2051), (5, 4096), (2, 5000), (3, 8192), (2, 16384), (3, 16391), (2, 40000)]


@gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(d)[6:] for d in t))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_norm_against_float64(types, shape):
    affine = ("both", "weight", "bias", "none")[(shape[0] + shape[1]) % 4]
    check(operands(shape, *types, affine, seed=shape[0] * 1000 + shape[1]), p=0.1, seed=1234567 + shape[1], offset=3)


@gpu
@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 255, 2047, 5000])
@pytest.mark.parametrize("cols", [8, 72, 256, 1000])
def test_norm_numbers_of_rows(rows, cols):
    """Rows that fill no workgroup, exactly one, several; sums of the parameters' gradients over one row and many."""
    check(operands((rows, cols), F32, F32, F32, "both", seed=rows + cols), p=0.2, seed=rows, offset=1)
    check(operands((rows, cols), BF16, None, F32, "both", seed=rows + cols + 1))


@gpu
@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 6, 7])
def test_norm_short_rows(cols):
    """Rows of fewer than eight elements, many of them, dense and apart, every type."""
    for k, types in enumerate(TYPES):
        rows = (1, 255, 257, 4000)[k % 4]
        o = operands((rows, cols), *types, ("both", "weight", "none")[k % 3], seed=cols * 10 + k)
        check(o, p=0.3, seed=k, offset=cols)
        wide = torch.full((rows, cols + 3), float("nan"), device="cuda", dtype=types[0])
        wide[:, 1:1 + cols] = o["x"]
        check(o, p=0.3, seed=k, offset=cols, x_view=wide[:, 1:1 + cols])


@gpu
@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
def test_norm_shapes_and_strides(affine):
    g = torch.Generator("cuda").manual_seed(2)
    base = torch.randn(6, 5, 300, device="cuda", generator=g)
    for view in (base[:, :, 20:276], base[:, :, 3:260], base[:, :, :250], base[:, 2, 1:258], base.transpose(0, 1)[..., :256], base.permute(2, 1, 0)[:64],
                 base[:1, :, 7:71].expand(4, 5, 64), base[3, 4, 10:266], base[::2, :, :128], base.flatten()[1:1 + 256 * 30].view(30, 256)):
        o = operands(tuple(view.shape), F32, None, F32, affine, seed=4)
        check(o, x_view=view)
        o = operands(tuple(view.shape), F32, F32, F32, affine, seed=5)
        wide = torch.randn(*view.shape[:-1], view.shape[-1] + 9, device="cuda", generator=g)
        o["residual"] = wide[..., 4:4 + view.shape[-1]]
        o["dy"] = o["dy"][..., :1].expand(view.shape)
        check(o, p=0.5, seed=8, offset=9, x_view=view)


@gpu
def test_norm_half_precision_unaligned():
    base = torch.randn(50 * 300 + 1, device="cuda", dtype=F16, generator=torch.Generator("cuda").manual_seed(3))
    for start in (0, 1):
        for cols in (256, 250):
            view = base[start:start + 50 * 300].view(50, 300)[:, 1:1 + cols]
            o = operands((50, cols), F16, F16, F16, "both", seed=6)
            check(o, p=0.25, seed=3, x_view=view)


@gpu
def test_norm_rows_of_special_values():
    """Constant rows, large offsets, and rows with infinities or NaN, which spoil their own results only."""
    x = torch.randn(40, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    x[3] = 5.0
    x[4] = 0.0
    x[5] += 1000.0
    x[6] *= 1e-20
    x[7] *= 1e12
    o = operands((40, 256), F32, None, F32, "both", seed=7)
    want, grads = check({**o, "x": x})
    assert torch.equal(layer_norm(x, o["weight"], o["bias"])[3:5], o["bias"].expand(2, 256))
    clean = layer_norm(x, o["weight"], o["bias"])
    x[10, 3], x[20, 100], x[30, 255] = float("inf"), float("nan"), float("-inf")
    y = layer_norm(x, o["weight"], o["bias"])
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[10, 20, 30]] = True
    assert torch.equal(y[~bad], clean[~bad]) and bool(y[bad].isnan().all())
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(layer_norm(leaf, o["weight"], o["bias"]), leaf, o["dy"])
    assert torch.equal(dx[~bad], grads["x"][~bad]) and bool(dx[bad].isnan().all())


@gpu
@pytest.mark.parametrize("cols", [5, 256, 257, 5000, 17000])
def test_norm_rows_beyond_the_range_of_fp32_are_nan(cols):
    x = torch.randn(6, cols, device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    clean = layer_norm(x)
    x[2] *= 1e25
    y = layer_norm(x)
    rest = [0, 1, 3, 4, 5]
    assert bool(y[2].isnan().all()) and torch.equal(y[rest], clean[rest])


@gpu
@pytest.mark.parametrize("cols", [256, 257])
def test_norm_beyond_32_bit_indexes(cols):
    """2.2e9 elements, 4.3 GB a tensor: rows at the far end and around 2^31 elements and bytes against the oracle."""
    rows, p, seed, offset = 2_200_000_000 // cols, 0.3, 99, 5
    g = torch.Generator("cuda").manual_seed(9)
    x, r, dy = (torch.empty(rows, cols, device="cuda", dtype=F16).normal_(generator=g) for _ in range(3))
    w, b = (torch.randn(cols, device="cuda", generator=g) for _ in range(2))
    y, mean, rstd = hip.norm_forward(x, w, b, 1e-5, r, p, seed, offset, want_stats=True)
    dx, dres, _, _ = hip.norm_backward(dy, x, mean, rstd, w, b, 1e-5, r, p, seed, offset, want=(True, True, False, False))
    for first in (0, 2 ** 30 // cols - 3, 2 ** 31 // cols - 3, rows - 6):
        part = slice(first, first + 6)
        factor = ref.keep((6, cols), p, seed, offset, first=first * cols).double() * ref.scale(p)
        want = ref.norm(x[part], w, b, 1e-5, r[part], factor, dy[part])
        tol = bounds(want, 1e-5, F16, F16, F32, ref.scale(p))
        for name, got in (("y", y), ("dx", dx), ("dresidual", dres)):
            within(got[part], want[name], tol[name], name)


@gpu
def test_join_drops_non_finite_values():
    x = torch.randn(16, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    m = ref.keep((16, 256), 0.5, 21, 2).cuda()
    r = torch.randn(16, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    want = dropout_add_layer_norm(torch.where(m, x, torch.zeros(())).contiguous(), r, p=0.5, seed=21, offset=2)
    spoiled = torch.where(m, x, torch.tensor([float("nan"), float("inf")], device="cuda").repeat(128))
    assert torch.equal(dropout_add_layer_norm(spoiled, r, p=0.5, seed=21, offset=2), want)


@gpu
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, F32), (F16, F32, F32)], ids=str)
@pytest.mark.parametrize("cols", [256, 250, 257])
def test_join_is_dropout_then_norm(types, cols):
    """One mask for the separate calls and the join; p = 0 and p = 1; the seed as a tensor."""
    o = operands((77, cols), *types, "both", seed=cols)
    args = o["x"], o["residual"], o["weight"], o["bias"]
    for p in (0.0, 0.3, 1.0):
        factor = ref.keep((77, cols), p, 5, 6).double() * ref.scale(p)
        assert torch.equal((dropout(torch.ones_like(o["x"]), p, 5, 6) != 0).cpu(), factor != 0)
        want = ref.norm(o["x"], o["weight"], o["bias"], 1e-5, o["residual"], factor)
        within(dropout_add_layer_norm(*args, p=p, seed=5, offset=6), want["y"], bounds(want, 1e-5, types[1], types[0], types[2])["y"], "y")
    a = dropout_add_layer_norm(*args, p=0.3, seed=5, offset=6)
    assert torch.equal(a, dropout_add_layer_norm(*args, p=0.3, seed=torch.tensor([5], device="cuda"), offset=6))


@gpu
def test_gradients_against_differences():
    """Directional derivatives of the float64 forward pass; tolerance: the bounds of the gradients, summed along the direction."""
    o = operands((23, 40), F32, F32, F32, "both", seed=11)
    p, seed, offset = 0.25, 31, 4
    want, grads = check(o, p=p, seed=seed, offset=offset)
    factor = ref.keep((23, 40), p, seed, offset).double() * ref.scale(p)
    tol = bounds(want, 1e-5, F32, F32, F32, ref.scale(p))
    g = torch.Generator().manual_seed(12)
    t = {k: o[k].double().cpu() for k in ("x", "residual", "weight", "bias")}
    loss = lambda t: float((ref.norm(t["x"], t["weight"], t["bias"], 1e-5, t["residual"], factor)["y"] * want["dy"]).sum())     # noqa: E731
    for k in t:
        v, h = torch.randn(t[k].shape, generator=g, dtype=torch.float64), 1e-6
        slope = (loss({**t, k: t[k] + h * v}) - loss({**t, k: t[k] - h * v})) / (2 * h)
        assert abs(slope - float((grads[k].double().cpu() * v).sum())) <= float((tol["d" + k] * v.abs()).sum()) + 1e-6


@gpu
def test_only_the_wanted_gradients():
    o = operands((30, 256), F32, F32, F32, "both", seed=13)
    names = ("x", "residual", "weight", "bias")
    full = None
    for wanted in (names, ("x",), ("residual",), ("weight",), ("bias",), ("x", "bias"), ("residual", "weight")):
        t = {k: o[k].detach().clone().requires_grad_(k in wanted) for k in names}
        y = dropout_add_layer_norm(*t.values(), p=0.1, seed=3, offset=1)
        y.backward(o["dy"])
        got = {k: t[k].grad for k in names}
        full = full or got
        for k in names:
            assert got[k] is None if k not in wanted else torch.equal(got[k], full[k])
    with torch.no_grad():
        assert not dropout_add_layer_norm(*t.values(), p=0.1, seed=3, offset=1).requires_grad


@gpu
def test_second_derivatives():
    """dropout is linear: its gradient's graph is its own; the normalisations refuse to build one."""
    x = torch.randn(4, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).requires_grad_()
    y = dropout(x, 0.5, 6) ** 2
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    second, = torch.autograd.grad(g.sum(), x)
    assert torch.equal(second.cpu(), ref.keep((4, 40), 0.5, 6, 0).float() * 8)
    for y in (layer_norm(x), dropout_add_layer_norm(x, x, p=0.5, seed=6)):
        with pytest.raises(hip.HipError, match="not differentiable"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


@gpu
def test_same_call_same_bits():
    o = operands((3000, 257), BF16, F32, F32, "both", seed=14)
    runs = []
    for _ in range(3):
        t = [o[k].detach().requires_grad_() for k in ("x", "residual", "weight", "bias")]
        y = dropout_add_layer_norm(*t, p=0.1, seed=3, offset=1)
        runs.append([y.detach(), *torch.autograd.grad(y, t, o["dy"])])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@gpu
def test_shared_weight_and_broadcast_inputs():
    """One weight used by two calls, a residual broadcast over rows: autograd adds the gradients up."""
    o = operands((12, 64), F32, F32, F32, "both", seed=15)
    w, b, row = o["weight"].requires_grad_(), o["bias"].requires_grad_(), o["residual"][:1].detach().clone().requires_grad_()
    y = layer_norm(dropout_add_layer_norm(o["x"], row.expand(12, 64), w, b, p=0.2, seed=1, offset=1), w, b)
    y.backward(o["dy"])
    factor = ref.keep((12, 64), 0.2, 1, 1).double() * ref.scale(0.2)
    first = ref.norm(o["x"], w, b, 1e-5, row.expand(12, 64), factor)
    second = ref.norm(first["y"], w, b, 1e-5, dy=o["dy"])
    first = ref.norm(o["x"], w, b, 1e-5, row.expand(12, 64), factor, second["dx"])
    # two chained operators, each off by less than 2^-24 * 100 of its results' size (D = 64)
    for got, want in ((w.grad, first["dweight"] + second["dweight"]), (b.grad, first["dbias"] + second["dbias"]), (row.grad, first["dresidual"].sum(0, keepdim=True))):
        assert float((got.double().cpu() - want).norm() / want.norm()) < 200 * E32


@gpu
def test_refusals():
    x = torch.zeros(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for call in (lambda: layer_norm(x.double()), lambda: layer_norm(x, w[:8]), lambda: layer_norm(x, w.half()), lambda: layer_norm(x.half(), w, w.half()),
                 lambda: layer_norm(x, w.cpu()), lambda: layer_norm(torch.ones((), device="cuda")), lambda: layer_norm(x[:, :0]), lambda: layer_norm(x, eps=0.0),
                 lambda: layer_norm(x, eps=-1.0), lambda: layer_norm(x, eps=float("nan")), lambda: dropout_add_layer_norm(x, x[:1]),
                 lambda: dropout_add_layer_norm(x, x.half()), lambda: dropout_add_layer_norm(x.half(), x.bfloat16()), lambda: dropout_add_layer_norm(x, x.cpu()),
                 lambda: dropout_add_layer_norm(x, x, p=1.1), lambda: dropout_add_layer_norm(x, x, p=0.1, offset=-1)):
        with pytest.raises(hip.HipError):
            call()
    y, mean, rstd = hip.norm_forward(x, w, w, want_stats=True)
    for bad in (dict(dy=y.half()), dict(dy=y[:2]), dict(mean=mean[:2]), dict(rstd=rstd.double())):
        with pytest.raises(hip.HipError):
            hip.norm_backward(**{**dict(dy=y, x=x, mean=mean, rstd=rstd, weight=w), **bad})


@gpu
def test_inputs_changed_between_the_passes_are_noticed():
    x, seed = torch.randn(8, 32, device="cuda").requires_grad_(), torch.tensor([4], device="cuda")
    y = dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_on_another_stream():
    side = torch.cuda.Stream()
    o = operands((500, 256), F32, F32, F32, "both", seed=16)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want, grads = check(o, p=0.1, seed=2)
    side.synchronize()


@gpu
def test_captured_step_draws_new_masks():
    """Forward and backward of both operators in one graph, the seed advanced inside it; every replay against eager calls, with eager
    work between the replays."""
    o = operands((300, 256), BF16, BF16, F32, "both", seed=17)
    seed = torch.tensor([100], device="cuda")
    keep = {}

    def step(seed):
        h = hip.dropout(o["x"], 0.2, seed, 1)
        y, mean, rstd = hip.norm_forward(h, o["weight"], o["bias"], 1e-5, o["residual"], 0.3, seed, 2, want_stats=True)
        dh, dres, dw, db = hip.norm_backward(o["dy"], h, mean, rstd, o["weight"], o["bias"], 1e-5, o["residual"], 0.3, seed, 2)
        return y, hip.dropout(dh, 0.2, seed, 1), dres, dw, db

    step(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed += 1
        keep["out"] = step(seed)
    for n in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in keep["out"]]
        want = step(100 + n)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
        torch.randn(1000, device="cuda").sum().item()


@gpu
def test_captured_autograd_step():
    """The same through autograd, captured with leaves of its own."""
    o = operands((64, 128), F32, F32, F32, "both", seed=18)
    seed = torch.tensor([7], device="cuda")
    leaves = [o[k].detach().clone().requires_grad_() for k in ("x", "residual", "weight", "bias")]
    eager = [t.detach().clone().requires_grad_() for t in leaves]

    def step(t, seed):
        y = dropout_add_layer_norm(*t, p=0.4, seed=seed, offset=5)
        return [y.detach(), *torch.autograd.grad(y, t, o["dy"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves, seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves, seed)
    for n in range(3):
        seed.fill_(50 + n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(eager, 50 + n))), n


@gpu
def test_capture_beside_a_living_eager_graph_is_refused():
    """An eager graph on the default stream holds the leaf's gradient node: a captured backward pass would wait on the default stream."""
    w = torch.ones(32, device="cuda").requires_grad_()
    x = torch.randn(4, 32, device="cuda")
    alive = layer_norm(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    out = None
    with torch.cuda.graph(graph):
        out = x + 1
        with pytest.raises(hip.HipError, match="eager graph"):
            layer_norm(x, w)
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer_norm(x, w).detach()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, layer_norm(x, w.detach()))


@gpu
def test_x_is_its_own_residual():
    o = operands((20, 48), F32, F32, F32, "both", seed=21)
    x = o["x"].clone().requires_grad_()
    dropout_add_layer_norm(x, x, o["weight"], o["bias"], p=0.5, seed=2, offset=3).backward(o["dy"])
    factor = ref.keep((20, 48), 0.5, 2, 3).double() * ref.scale(0.5)
    want = ref.norm(o["x"], o["weight"], o["bias"], 1e-5, o["x"], factor, o["dy"])
    tol = bounds(want, 1e-5, F32, F32, F32, 2.0)
    within(x.grad, want["dx"] + want["dresidual"], tol["dx"] + tol["dresidual"] + u(F32) * (want["dx"] + want["dresidual"]).abs(), "dx")


@gpu
def test_backward_again():
    o = operands((20, 48), F32, F32, F32, "both", seed=22)
    x = o["x"].clone().requires_grad_()
    y = dropout_add_layer_norm(x, o["residual"], o["weight"], o["bias"], p=0.5, seed=2)
    a, = torch.autograd.grad(y, x, o["dy"], retain_graph=True)
    b, = torch.autograd.grad(y, x, o["dy"])
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, o["dy"])


@gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_block(reentrant):
    """The mask is an argument's function, so a recomputed forward pass draws it again: the same bits as without a checkpoint."""
    from torch.utils.checkpoint import checkpoint
    o = operands((50, 256), F16, F32, F32, "both", seed=23)

    def block(x, r, w, b):
        return layer_norm(dropout_add_layer_norm(dropout(x, 0.2, 5, 1), r, w, b, p=0.3, seed=5, offset=2), w, b)

    results = []
    for how in ("plain", "checkpoint"):
        t = [o[k].detach().clone().requires_grad_() for k in ("x", "residual", "weight", "bias")]
        y = block(*t) if how == "plain" else checkpoint(block, *t, use_reentrant=reentrant)
        y.backward(o["dy"])
        results.append([y.detach()] + [v.grad for v in t])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
def test_saved_tensors_elsewhere():
    o = operands((50, 257), BF16, None, F32, "both", seed=24)
    results = []
    for hooks in (False, True):
        x = o["x"].clone().requires_grad_()
        if hooks:
            with torch.autograd.graph.save_on_cpu():
                y = layer_norm(x, o["weight"], o["bias"])
        else:
            y = layer_norm(x, o["weight"], o["bias"])
        results.append(torch.autograd.grad(y, x, o["dy"])[0])
    assert torch.equal(*results)


@gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwAD
    x = torch.randn(4, 16, device="cuda")
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda: layer_norm(d), lambda: dropout(d, 0.5, 1), lambda: dropout_add_layer_norm(x, d)):
            with pytest.raises(hip.HipError, match="forward-mode"):
                call()


@gpu
def test_two_host_threads():
    import threading
    failed = []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(8):
                    check(operands((64 + seed, 130 + k), F32, F32, F32, "both", seed=seed * 100 + k), p=0.25, seed=k, offset=seed)
        except BaseException as e:      # noqa: B902
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_the_current_one():
    o = operands((64, 256), F32, F32, F32, "both", seed=25)
    there = {k: v.to("cuda:1") for k, v in o.items()}
    torch.cuda.synchronize(0)
    torch.cuda.synchronize(1)
    check(there, p=0.25, seed=3)
    with pytest.raises(hip.HipError):
        dropout_add_layer_norm(there["x"], o["residual"])


@gpu
def test_block_of_the_tracker_trains():
    """A feed-forward block as the tracker has it -- norm(x + dropout(attn)), norm2(x + dropout(linear(dropout(gelu(linear(x)))))) -- with all
    gradients, against float64 autograd with the same masks.  The products run in float64 here, so what is off is the operators' own:
    six of them, each below 2^-24 * 150 of its result's norm (D = 1024 at most), chained through factors near one."""
    g = torch.Generator().manual_seed(19)
    R, D, H, p, seed = 96, 256, 1024, 0.1, 2024
    t = {k: torch.randn(*s, generator=g) * c for k, s, c in (("x", (R, D), 1), ("attn", (R, D), 1), ("w1", (H, D), D ** -0.5), ("w2", (D, H), H ** -0.5),
                                                              ("n1", (D,), 1), ("b1", (D,), 1), ("n2", (D,), 1), ("b2", (D,), 1))}
    dy = torch.randn(R, D, generator=g)
    a = {k: v.cuda().requires_grad_() for k, v in t.items()}
    lin = lambda x, w: (x.double() @ w.double().t()).float()     # noqa: E731
    h = dropout_add_layer_norm(a["attn"], a["x"], a["n1"], a["b1"], p=p, seed=seed, offset=0)
    f = lin(dropout(torch.nn.functional.gelu(lin(h, a["w1"]).double()).float(), p, seed, 1), a["w2"])
    y = layer_norm(dropout(f, p, seed, 2) + h, a["n2"], a["b2"])
    y2 = dropout_add_layer_norm(f, h, a["n2"], a["b2"], p=p, seed=seed, offset=2)
    y2.backward(dy.cuda())
    b = {k: v.double().requires_grad_() for k, v in t.items()}
    fac = [ref.keep(s, p, seed, k).double() * ref.scale(p) for k, s in enumerate(((R, D), (R, H), (R, D)))]
    ln = lambda z, w, c: torch.nn.functional.layer_norm(z, (D,), w, c, 1e-5)     # noqa: E731
    h64 = ln(b["x"] + b["attn"] * fac[0], b["n1"], b["b1"])
    f64 = (torch.nn.functional.gelu(h64 @ b["w1"].t()) * fac[1]) @ b["w2"].t()
    y64 = ln(h64 + f64 * fac[2], b["n2"], b["b2"])
    y64.backward(dy.double())
    off = lambda got, want: float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())     # noqa: E731
    assert off(y, y64) < 1000 * E32 and off(y2, y64) < 1000 * E32
    for k in t:
        assert off(a[k].grad, b[k].grad) < 1000 * E32, (k, off(a[k].grad, b[k].grad))


# ---------------------------------------------------------------------------------------------- rows far from zero

def offset_bounds(o, eps, dtype, depth=None):
    """Tolerances where the mean is far larger than the spread (types: all `dtype`, parameters fp32, z exact in fp32).  depth as above.
    The first mean is off by delta <= e (depth + 2) mean|z|; the deviations from it are off by e of themselves; their mean, by which they are
    corrected, by e (depth + 3) mean|z - first| <= e (depth + 3) (delta + MAD); the variance by e (depth + 8) (var + delta^2).  So
      E = e rstd ((depth + 8) (delta + MAD) + 2 |z - mean|) + e (depth + 16) |xhat| (1 + delta^2 / (var + eps))
    of which only e^2 mean|z| grows with the offset.  The backward pass takes z from the stored mean, an fp32 number:
      Eb = E + e |mean| rstd,  and from there the module's formulas."""
    D = o["z"].shape[-1]
    depth = depth or 8 * math.ceil(D / 2048) + 32
    mean = lambda t: t.mean(-1, keepdim=True)        # noqa: E731
    dev = (o["z"] - o["mean"]).abs()
    delta = E32 * (depth + 2) * mean(o["z"].abs())
    E = E32 * o["rstd"] * ((depth + 8) * (delta + mean(dev)) + 2 * dev) + E32 * (depth + 16) * o["xhat"].abs() * (1 + (delta * o["rstd"]) ** 2)
    t = {"y": u(dtype) * o["y"].abs() + o["w"].abs() * E + 4 * E32 * ((o["xhat"] * o["w"]).abs() + o["b"].abs()) + tiny(dtype),
         "mean": E32 * o["mean"].abs() + E32 * (depth + 3) * (delta + mean(dev)),
         "rstd": E32 * (depth + 16) * o["rstd"] * (1 + (delta * o["rstd"]) ** 2)}
    Eb = E + E32 * o["mean"].abs() * o["rstd"]
    g, xh, dz = o["g"].abs(), o["xhat"].abs() + Eb, o["dresidual"].abs()
    raw = o["rstd"] * (4 * E32 * g + E32 * (depth + 4) * mean(g) + xh * (E32 * (depth + 4) * mean(g * xh) + mean(g * Eb)) + Eb * o["c2"].abs()) \
        + E32 * (depth + 16) * (1 + (delta * o["rstd"]) ** 2) * dz
    rows = o["z"].numel() // D
    n = min(rows, rows / 64 + 64) + 32
    flat = lambda v: v.reshape(-1, D).sum(0)         # noqa: E731
    t["dx"] = t["dresidual"] = u(dtype) * dz + raw + tiny(dtype)
    t["dweight"] = u(F32) * o["dweight"].abs() + flat(o["dy"].abs() * Eb) + E32 * n * flat(o["dy"].abs() * xh)
    return t


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [5, 257, 768, 1000, 1537, 5000, 17000])
def test_norm_rows_far_from_zero(dtype, cols):
    """Constant rows, rows that are constant but for one element, and small spreads on large offsets: what is left is the spread's, whatever the
    offset is; layer_norm and the join (whose sum is exact here: the residual holds the other half)."""
    offsets = [1000.0, 1000.1, 65504.0, 30000.3, -12345.6, 0.1, 3.0]
    rows = torch.tensor(offsets).repeat_interleave(3)[:, None].repeat(1, cols)
    step = torch.finfo(dtype).eps * torch.tensor(offsets).abs()
    for i in range(len(offsets)):
        rows[3 * i + 1, cols // 3] -= 2 * step[i]                                     # one element two steps lower
        rows[3 * i + 2] -= 4 * step[i] * torch.randint(0, 3, (cols,), generator=torch.Generator().manual_seed(i)) * torch.sign(rows[3 * i + 2])
    g = torch.Generator().manual_seed(cols)
    w, b = 1 + 0.2 * torch.randn(cols, generator=g), 0.2 * torch.randn(cols, generator=g)
    dy = torch.randn(*rows.shape, generator=g).to(dtype)
    x = rows.to(dtype)
    for joined in (False, True):
        half = (x.float() / 2).to(dtype) if joined else x                              # exact: a power of two
        r = half if joined else None
        want = ref.norm(half, w, b, 1e-5, r, None, dy)
        tol = offset_bounds(want, 1e-5, dtype)
        dev = lambda t: None if t is None else t.cuda()                                # noqa: E731
        y, mean, rstd = hip.norm_forward(dev(half), dev(w), dev(b), 1e-5, dev(r), want_stats=True)
        within(y, want["y"], tol["y"], "y")
        within(mean[:, None], want["mean"], tol["mean"], "mean")
        within(rstd[:, None], want["rstd"], tol["rstd"], "rstd")
        dx, dres, dw, _ = hip.norm_backward(dev(dy), dev(half), mean, rstd, dev(w), dev(b), 1e-5, dev(r))
        within(dx, want["dx"], tol["dx"], "dx")
        if joined:
            within(dres, want["dresidual"], tol["dresidual"], "dresidual")
        within(dw, want["dweight"], tol["dweight"], "dweight")


@gpu
def test_norm_constant_rows_at_small_eps():
    """No eps makes something of the rounding of a constant row: below 2^-18 of the squares that the first mean leaves, a variance is noise."""
    x = torch.tensor([1000.1, -30000.3, 0.1])[:, None].repeat(1, 1000).cuda()
    for eps in (1e-5, 1e-12, 1e-30, 1.2e-38):
        assert float(layer_norm(x, eps=eps).abs().max()) < 2 ** 9 * E32 * 64, eps


# ---------------------------------------------------------------------------------------------- sizes beyond one launch

def test_grids_stay_below_what_a_launch_holds(tmp_path):
    """launch.hpp, compiled by itself: HIP takes fewer than 2^32 threads along a dimension."""
    import os
    import subprocess
    src, lib = tmp_path / "launch.cpp", tmp_path / "launch.so"
    src.write_text('#include "launch.hpp"\nextern "C" unsigned grid(long long want, int threads) { return lbm::grid_of(want, threads); }\n')
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lbm_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", csrc, str(src), "-o", str(lib)], check=True)
    grid = C.CDLL(str(lib)).grid
    grid.argtypes, grid.restype = [C.c_longlong, C.c_int], C.c_uint
    for threads in (64, 192, 256, 1024):
        for want in (1, 255, 1 << 22, (1 << 24) - 1, 1 << 24, 1 << 26, 1 << 30, 1 << 40):
            g = grid(want, threads)
            assert 1 <= g <= want and g * threads < 1 << 32
            assert g == want or (g + 1) * threads >= 1 << 32


@gpu
def test_dropout_beyond_one_launch():
    """2^35 elements are 2^32 threads' work: the last chunks are a thread's second."""
    n, p, seed, offset = (1 << 35) + 4099, 0.25, 42, 7
    lib = hip.load()
    torch.cuda.empty_cache()
    x = torch.ones(n, device="cuda", dtype=F16)
    assert lib.lbm_hip_dropout(x.data_ptr(), x.data_ptr(), n, 1, p, seed, None, offset, torch.cuda.current_stream().cuda_stream) == 0, lib.lbm_hip_last_error()
    for first in (0, (1 << 32) - 1000, (1 << 35) - 3048, n - 2000):
        got = x[first:first + 2000].float().cpu()
        want = ref.keep((2000,), p, seed, offset, first=first)
        assert torch.equal(got != 0, want) and torch.equal(got[want], torch.full((int(want.sum()),), ref.scale(p)).half().float())
    del x
    torch.cuda.empty_cache()


@gpu
def test_norm_forward_beyond_one_launch():
    """2^32 rows of two columns and some: the last ones belong to a second launch.  With statistics of every row: 34 GB."""
    rows, cols, p, seed, offset = (1 << 32) + 1003, 2, 0.3, 11, 4
    torch.cuda.empty_cache()
    g = torch.Generator("cuda").manual_seed(10)
    x = torch.empty(rows, cols, device="cuda", dtype=F16)
    x.view(-1)[:1 << 20].normal_(generator=g)
    n = 1 << 20
    while n < x.numel():                                                              # a pattern of 2^20 numbers over all of it
        k = min(n, x.numel() - n)
        x.view(-1)[n:n + k] = x.view(-1)[:k]
        n += k
    w, b = torch.tensor([1.25, -0.5], device="cuda"), torch.tensor([0.1, 0.2], device="cuda")
    y, mean, rstd = hip.norm_forward(x, w, b, 1e-5, x, p, seed, offset, want_stats=True)
    edge = ((1 << 24) - 1) * 256
    for first in (0, (1 << 31) - 3, edge - 500, rows - 1000):
        part = slice(first, first + 1000)
        factor = ref.keep((1000, cols), p, seed, offset, first=first * cols).double() * ref.scale(p)
        want = ref.norm(x[part], w, b, 1e-5, x[part], factor)
        within(y[part], want["y"], bounds(want, 1e-5, F16, F16, F32, ref.scale(p))["y"], "y")
        within(mean[part][:, None], want["mean"], 4 * E32 * (want["z"].abs() + want["xs"].abs()).mean(-1, keepdim=True) + 2.0 ** -140, "mean")
    del x, y, mean, rstd
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("bias", [True, False])
def test_norm_columns_beyond_one_launch(bias):
    """2^26 columns and some: their sums are 2^32 threads' work.  dy is zero but for a few columns, so that the oracle's sums are short."""
    rows, cols = 2, (1 << 26) + 4001
    g = torch.Generator("cuda").manual_seed(12)
    x = torch.empty(rows, cols, device="cuda", dtype=F16).normal_(generator=g)
    w = torch.ones(cols, device="cuda", dtype=F16)
    dy = torch.zeros(rows, cols, device="cuda", dtype=F16)
    at = torch.tensor([0, 5, (1 << 25) + 3, (1 << 26) - 1, 1 << 26, cols - 1], device="cuda")
    dy[:, at] = torch.randn(rows, len(at), device="cuda", generator=g).half()
    # statistics that are given, not computed: what is checked is the sums over rows
    mean, rstd = torch.tensor([0.25, -0.5], device="cuda"), torch.tensor([1.5, 0.75], device="cuda")
    _, _, dw, db = hip.norm_backward(dy, x, mean, rstd, w, w if bias else None, want=(False, False, True, bias))
    term = dy[:, at].double() * (x[:, at].double() - mean[:, None].double()) * rstd[:, None].double()
    want = torch.zeros(cols, device="cuda", dtype=torch.float64)
    want[at] = term.sum(0)
    tol = torch.zeros_like(want)
    tol[at] = u(F16) * want[at].abs() + 8 * E32 * term.abs().sum(0) + tiny(F16)
    within(dw, want.cpu(), tol.cpu(), "dweight")
    if bias:
        want[at] = dy[:, at].double().sum(0)
        tol[at] = u(F16) * want[at].abs() + 8 * E32 * dy[:, at].double().abs().sum(0) + tiny(F16)
        within(db, want.cpu(), tol.cpu(), "dbias")
    else:
        assert db is None


# ---------------------------------------------------------------------------------------------- the host path

def test_cpu_tensors_that_want_gradients_are_refused():
    """The documented error, also where the machine has no GPU to be asked."""
    x, w = torch.zeros(2, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    for call in (lambda: layer_norm(x), lambda: layer_norm(x, w, w), lambda: layer_norm(x.detach(), w), lambda: dropout(x, 0.5, 1),
                 lambda: dropout_add_layer_norm(x, x, w), lambda: dropout_add_layer_norm(x.detach(), x)):
        with pytest.raises(hip.HipError, match="GPU"):
            call()


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_capture_on_a_device_that_is_not_the_current_one():
    """The refusal beside a living eager graph asks the stream of x's device, whichever device is current."""
    w = torch.ones(32, device="cuda:1").requires_grad_()
    x = torch.randn(4, 32, device="cuda:1")
    alive = layer_norm(x, w)
    torch.cuda.synchronize(1)
    side = torch.cuda.Stream(device="cuda:1")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.device(1), torch.cuda.stream(side):
        graph.capture_begin()
        out = x + 1
        with torch.cuda.device(0), pytest.raises(hip.HipError, match="eager graph"):
            layer_norm(x, w)
        graph.capture_end()
    del alive, out


@gpu
@pytest.mark.parametrize("joined", [False, True])
def test_saved_tensors_that_come_back_different_are_refused(joined):
    """Hooks that change size, type or device: the backward pass would read dy in another type or beyond its end."""
    def run(unpack):
        x, r, w = torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda"), torch.ones(40, device="cuda")
        x.requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = dropout_add_layer_norm(x, r, w, p=0.2, seed=1) if joined else layer_norm(x, w)
        return torch.autograd.grad(y, x, torch.ones_like(y))

    run(lambda t: t.clone())
    changes = [lambda t: t.half(), lambda t: torch.cat([t, t]), lambda t: t.cpu(), lambda t: t[..., :20], lambda t: t[:3], lambda t: t.half() if t.dim() == 1 else t,
               lambda t: t[:20] if t.dim() == 1 else t, lambda t: t.double()]
    for k, change in enumerate(changes):
        with pytest.raises(hip.HipError):
            run(change)


@gpu
def test_saved_seeds_that_come_back_different_are_refused():
    x, seed = torch.randn(6, 40, device="cuda").requires_grad_(), torch.tensor([3], device="cuda")
    for call in (lambda: dropout(x, 0.5, seed), lambda: dropout_add_layer_norm(x, x, p=0.5, seed=seed)):
        for change in (lambda t: t.cpu(), lambda t: t.int(), lambda t: t.expand(2)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == torch.int64 else t):
                y = call()
            with pytest.raises(hip.HipError, match="seed"):
                torch.autograd.grad(y, x, torch.ones_like(y))


@gpu
def test_function_transforms_and_sparse_tensors_are_refused():
    """torch.func's wrappers and sparse tensors have no memory to hand to a kernel: an error that says so, for operands and gradients."""
    x, w = torch.randn(3, 4, 16, device="cuda"), torch.ones(16, device="cuda")
    f = torch.func
    for call in (lambda: f.vmap(layer_norm)(x), lambda: f.vmap(lambda v: dropout(v, 0.5, 1))(x), lambda: f.vmap(lambda v: dropout_add_layer_norm(v, v))(x),
                 lambda: f.grad(lambda v: layer_norm(v).sum())(x), lambda: f.grad(lambda v: dropout(v, 0.5, 1).sum())(x),
                 lambda: f.grad(lambda v: layer_norm(x, v).sum())(w), lambda: f.vmap(lambda v: layer_norm(x, v))(torch.stack([w, w])),
                 lambda: f.vmap(lambda v: hip.norm_forward(v, None, None))(x), lambda: dropout(x.to_sparse(), 0.5, 1), lambda: layer_norm(x[0].to_sparse())):
        with pytest.raises(hip.HipError, match="plain dense tensor"):
            call()
    for op in (lambda t: layer_norm(t), lambda t: dropout(t, 0.5, 1)):
        leaf = x[0].clone().requires_grad_()
        y = op(leaf)
        with pytest.raises(hip.HipError, match="plain dense tensor"):
            torch.nn.functional.embedding(torch.tensor([0, 2], device="cuda"), y, sparse=True).sum().backward()
    with pytest.raises(hip.HipError, match="seed"):
        f.vmap(lambda s: dropout(x, 0.5, s))(torch.arange(3, device="cuda"))


@gpu
def test_negative_views():
    """The imaginary part of a conjugate is a view that torch negates when it is read."""
    g = torch.Generator("cuda").manual_seed(31)
    bits = lambda *shape: torch.randn(*shape, dtype=torch.complex64, device="cuda", generator=g).conj().imag.as_strided(shape, torch.empty(shape).stride())     # noqa: E731
    x, r, w, b, dy = bits(6, 40), bits(6, 40), bits(40), bits(40), bits(6, 40)
    assert all(t.is_neg() and t.is_contiguous() for t in (x, r, w, b, dy))
    plain = [t.resolve_neg() for t in (x, r, w, b)]
    assert torch.equal(dropout(x, 0.4, 3, 1), dropout(plain[0], 0.4, 3, 1))
    assert torch.equal(layer_norm(x[0:1, 4:], w[4:], b[4:]), layer_norm(plain[0][0:1, 4:], plain[2][4:], plain[3][4:]))
    results = []
    for t, d in (((x, r, w, b), dy), (plain, dy.resolve_neg())):
        leaves = [v.detach().requires_grad_() for v in t]
        y = dropout_add_layer_norm(*leaves, p=0.3, seed=2)
        results.append([y.detach(), *torch.autograd.grad(y, leaves, d)])
    assert all(torch.equal(p, q) for p, q in zip(*results))
    leaf = plain[0].detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(dropout(leaf, 0.4, 3), leaf, dy)[0], dropout(dy.resolve_neg(), 0.4, 3))


# ---------------------------------------------------------------------------------------------- very long sums

@gpu
@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("offset", [0.0, 500.0])
def test_norm_sums_of_millions_of_columns(offset, joined):
    """Equal terms round alike, so that a long chain of fp32 additions drifts instead of averaging out: rows of +-1.0001, dy of 1.0003.  A sum's fp32
    additions are eight of a chunk, a tree over 64 lanes and four waves: depth 32, however long the row is."""
    cols = 4_000_003
    x = (torch.arange(cols) % 2 * 2 - 1).float()[None] * torch.tensor([[1.0001], [0.7003]]) + offset
    dy = torch.full((2, cols), 1.0003)
    dy[:, ::3] = 0.5001
    r = x / 2 if joined else None
    x = x / 2 if joined else x                                                         # the join adds the halves up again, exactly
    want = ref.norm(x, None, None, 1e-5, r, None, dy)
    tol = offset_bounds(want, 1e-5, F32, depth=32)
    r = None if r is None else r.cuda()
    y, mean, rstd = hip.norm_forward(x.cuda(), None, None, 1e-5, r, want_stats=True)
    within(mean[:, None], want["mean"], tol["mean"], "mean")
    within(rstd[:, None], want["rstd"], tol["rstd"], "rstd")
    within(y, want["y"], tol["y"], "y")
    dx, dres, _, _ = hip.norm_backward(dy.cuda(), x.cuda(), mean, rstd, None, None, 1e-5, r)
    within(dx, want["dx"], tol["dx"], "dx")
    if joined:
        within(dres, want["dresidual"], tol["dresidual"], "dresidual")


@gpu
@pytest.mark.parametrize("cols,rows", [(16392, 200003), (2_100_001, 1603)])
def test_norm_wide_column_sums_of_many_rows(cols, rows):
    """Equal terms again: every row the same, dy of 1.0003 and xhat near 0.7.  A column's fp32 additions are at most 64 rows in a thread and 64 partial
    sums (32 slices of at most 32); what 64 rows make is added up in fp64."""
    torch.cuda.empty_cache()
    x = torch.empty(rows, cols, device="cuda", dtype=F16)
    x.copy_((torch.arange(cols, device="cuda") % 7 * 0.03 + 0.9).half().expand(rows, cols))
    dy = torch.full((rows, cols), 1.0003, device="cuda").half() if rows * cols < 1 << 30 else torch.empty(rows, cols, device="cuda", dtype=F16).fill_(1.0003)
    mean, rstd = torch.full((rows,), 0.25, device="cuda"), torch.full((rows,), 0.8001, device="cuda")
    w = torch.ones(cols, device="cuda")
    _, _, dw, db = hip.norm_backward(dy, x, mean, rstd, w, w, want=(False, False, True, True))
    d, xhat = dy[0].double().cpu(), (x[0].double().cpu() - 0.25) * rstd[0].double().cpu()
    del x, dy
    torch.cuda.empty_cache()
    within(dw, rows * d * xhat, E32 * (64 + 64 + 6) * rows * d * xhat, "dweight")
    within(db, rows * d, E32 * (64 + 64 + 2) * rows * d, "dbias")


def test_no_kernel_that_no_call_reaches():
    """Teams of a wave hold four chunks a lane only in layer_norm's forward pass (1537 .. 2048 columns), and the join's two chunks a lane are never loaded
    dword by dword: kernels for the other cases would only make the library larger."""
    import os
    import re
    blob = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lbm_amd", "liblbm_hip.so"), "rb").read()
    found = {m.group(0) for m in re.finditer(rb"_ZN3lbm15norm_(bwd|fwd)_kernelI[A-Za-z0-9_]+NS_8LoadModeE[0-9]EEEv", blob)}
    assert len(found) > 40
    fwd = [m for m in found if b"norm_fwd" in m]
    for m in found - set(fwd):
        assert not re.search(rb"Li4ELNS_8LoadMode", m), m                              # <TX, TR, RES, K, MODE>
    for m in fwd:                                                                      # <TX, TR, RES, K, U, MODE>
        assert not re.search(rb"Li1ELi4ELi\dELNS_8LoadMode", m) and not re.search(rb"Li1ELi2ELi\dELNS_8LoadModeE1E", m), m


# ---------------------------------------------------------------------------------------------- several rows a team, a workgroup, a launch

MANY = [  # rows just above a threshold and no multiple of it; columns; types
    # forward in a wave: four (K = 1) and two (K = 2, 3) rows in flight a team, from teams * U * 2048 rows on; backward: 16 rounds of a workgroup
    (65536 + 13, 256, (F16, None, F32)), (65536 + 13, 253, (BF16, None, BF16)), (131072 + 5, 136, (F32, None, F32)), (131072 + 5, 135, (F16, None, F16)),
    (16384 + 3, 1000, (BF16, None, F32)), (16384 + 3, 1001, (F16, None, F32)), (16384 + 5, 1048, (F16, None, F32)), (5000, 2047, (BF16, None, F32)),
    (32768 + 9, 250, (F16, F32, F32)), (32768 + 9, 249, (BF16, BF16, BF16)), (9001, 1021, (F16, F16, F32)), (6000, 1536, (BF16, F32, F32)), (262144 + 77, 5, (F16, F32, F32)),
    # forward in a workgroup: more than 256 (1024 / threads) rows, so that a second and a third row meet the loads ahead and the sums' memory;
    # backward: more than two rows a workgroup, one, two (rows >= 4096) and three (>= 6144) workgroups a CU
    (1300, 2051, (F16, None, F32)), (2900, 2051, (F32, F32, F32)), (4200, 2051, (BF16, BF16, F32)), (6200, 1537, (BF16, None, F32)), (6200, 1544, (F16, F32, F32)),
    (800, 4104, (F32, None, F32)), (1101, 4099, (BF16, BF16, BF16)), (600, 8192, (F16, None, F16)), (821, 8191, (BF16, F32, F32)),
    (600, 16384, (BF16, None, F32)), (777, 16383, (F16, None, F32)), (600, 16384, (F32, None, F32)), (600, 16377, (F16, F16, F32)), (520, 9000, (F32, F32, F32)),
    # beyond 16384 columns: several rounds of a workgroup in the column sums
    (1100, 17001, (BF16, F32, F32)),
]


@gpu
@pytest.mark.parametrize("rows,cols,types", MANY, ids=lambda v: "-".join(str(d)[6:] for d in v) if isinstance(v, tuple) else str(v))
def test_norm_many_rows_against_float64(rows, cols, types):
    check(operands((rows, cols), *types, "both", seed=rows + cols), p=0.15, seed=rows, offset=cols)


@gpu
@pytest.mark.parametrize("cols", [256, 257, 2051, 20001])
def test_norm_column_sums_beyond_32_bit_indexes(cols):
    """4.4e9 elements: dy is zero but in a few rows at both ends and around 2^31 and 2^32 elements, so that the oracle's sums are short."""
    rows, p, seed, offset = 4_400_000_000 // cols, 0.3, 99, 5
    torch.cuda.empty_cache()
    g = torch.Generator("cuda").manual_seed(cols)
    x = torch.empty(rows, cols, device="cuda", dtype=F16).normal_(generator=g)
    dy = torch.zeros(rows, cols, device="cuda", dtype=F16)
    at = [0, 1, 2 ** 31 // cols - 1, 2 ** 31 // cols, 2 ** 32 // cols - 1, 2 ** 32 // cols, 2 ** 32 // cols + 1, rows - 2, rows - 1]
    for r in at:
        dy[r] = torch.randn(cols, device="cuda", generator=g).half()
    w = torch.randn(cols, device="cuda", generator=g)
    _, mean, rstd = hip.norm_forward(x, w, w, 1e-5, x, p, seed, offset, want_stats=True)
    _, _, dw, db = hip.norm_backward(dy, x, mean, rstd, w, w, 1e-5, x, p, seed, offset, want=(False, False, True, True))
    factor = torch.cat([ref.keep((1, cols), p, seed, offset, first=r * cols) for r in at]).double() * ref.scale(p)
    want = ref.norm(x[at], w, w, 1e-5, x[at], factor, dy[at])
    tol = bounds(want, 1e-5, F16, F16, F32, ref.scale(p))
    within(dw, want["dweight"], tol["dweight"], "dweight")
    within(db, want["dbias"], tol["dbias"], "dbias")
    del x, dy
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------- the build

def _plan(*args):
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lbm_amd", "csrc")
    return subprocess.run(["make", "-n", "-C", csrc, *args], check=True, capture_output=True, text=True).stdout


def test_the_library_builds_without_torch():
    """The C interface needs no torch: only the host path of the training operators is left out, and make says so."""
    with_torch, without = _plan("-B", "all"), _plan("-B", "all", "PYTHON=/bin/false")
    assert "torch_ops.cpp" in with_torch and "is not built" not in with_torch
    assert "torch_ops.cpp" not in without and "is not built" in without
    for plan in (with_torch, without):
        assert "norm_bwd.hip" in plan and "-o ../liblbm_hip.so" in plan


def test_the_host_path_is_rebuilt_for_another_torch():
    import os
    version = os.path.join(os.path.dirname(torch.__file__), "version.py")
    assert "torch_ops.cpp" in _plan("-W", version, "all")


def test_build_compiles_what_is_built_already(monkeypatch):
    """build() is the check that every source compiles: it may not stop at a library that is there."""
    import subprocess

    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    entry.build()
    monkeypatch.undo()
    plan = subprocess.run([*calls[0], "-n"], check=True, capture_output=True, text=True).stdout
    assert "norm_bwd.hip" in plan and "gemm.hip" in plan and "torch_ops.cpp" in plan


@gpu
def test_batched_gradients_are_refused():
    """is_grads_batched maps the backward pass with vmap: gradients without memory of their own."""
    x, w = torch.randn(5, 24, device="cuda").requires_grad_(), torch.ones(24, device="cuda").requires_grad_()
    for y in (layer_norm(x, w), dropout(x, 0.5, 1), dropout_add_layer_norm(x, x.detach(), w, p=0.5, seed=torch.tensor([4], device="cuda"))):
        with pytest.raises(hip.HipError, match="plain dense tensor"):
            torch.autograd.grad(y, x, torch.ones(2, 5, 24, device="cuda"), is_grads_batched=True)


@gpu
@pytest.mark.filterwarnings("ignore")
def test_inside_a_compiled_function():
    """torch.compile leaves the operators outside of its graphs: the same bits, gradients too."""
    o = operands((40, 136), F32, F32, F32, "both", seed=41)

    def block(x, r, w, b):
        return layer_norm(torch.sin(dropout_add_layer_norm(dropout(x * 2, 0.2, 5, 1), r, w, b, p=0.3, seed=5, offset=2)) + r, w, b)

    results = []
    for f in (block, torch.compile(block, backend="eager")):
        t = [o[k].detach().clone().requires_grad_() for k in ("x", "residual", "weight", "bias")]
        y = f(*t)
        results.append([y.detach(), *torch.autograd.grad(y, t, o["dy"])])
    assert all(torch.equal(p, q) for p, q in zip(*results))


@gpu
@pytest.mark.parametrize("op", [lambda t: layer_norm(t), lambda t: dropout(t, 0.5, 1), lambda t: dropout_add_layer_norm(t.detach(), t, p=0.5, seed=2)],
                         ids=["layer_norm", "dropout", "join"])
def test_captured_backward_into_an_eager_graph_is_refused(op):
    """x is the result of an eager operation on the default stream: a captured backward pass would make that stream wait inside the capture.  Captured
    without its backward pass, or with all of the graph inside, it runs."""
    leaf = torch.randn(4, 32, device="cuda").requires_grad_()
    x = leaf * 2
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = op(x)
        with pytest.raises(hip.HipError, match="eager graph"):
            torch.autograd.grad(y, leaf, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.detach(), op(x.detach()))
    del x, y
    torch.cuda.synchronize()
    inside = leaf.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = op(inside * 2)
        d, = torch.autograd.grad(y, inside, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    y = op(leaf * 2)
    assert torch.equal(d, torch.autograd.grad(y, leaf, torch.ones_like(y))[0])


@gpu
@pytest.mark.parametrize("cols", [3, 1030, 1700, 2051, 8200, 16384, 17001])
def test_norm_without_rows(cols):
    """Every kernel's form of no work at all: empty results, zeros as the parameters' gradients."""
    for types in ((F32, None, F32), (F16, None, F16), (BF16, F32, F32)):
        o = operands((0, cols), *types, "both", seed=cols)
        _, grads = check(o, p=0.2, seed=1)
        assert not grads["weight"].any() and not grads["bias"].any()
    x = torch.zeros(2, 0, cols, device="cuda", requires_grad=True)
    assert layer_norm(x).shape == (2, 0, cols) and dropout(x, 0.5, 1).shape == (2, 0, cols)
