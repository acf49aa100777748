"""LayerNorm and the linear layer with their gradients, and 8-bit checkpoints, against the formulas in 64 bits.

Tolerances count roundings.  U = 2^-24 is fp32's; ``half`` is that of the output's type.  Sums of c terms in fp32 are off by at
most their depth times U of the sum of magnitudes; the tensor core's accumulation is given 2 U a term, since it may cut off
instead of rounding; an activation or its slope 16 U of its argument or of one (the error function's and the exponential's few
units in the last place, and 1 + erf for arguments far below zero)."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a step of subnormals, and as much again


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def check(name, got, want, bound):
    import bioemu2_b200._lib as L

    assert L.device_status() == 0
    got = got.double()
    assert got.shape == want.shape, name
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off by up to {float(((got - want).abs() / bound).max()):.3g} bounds; "
                           f"first {got[bad][:3].tolist()} want {want[bad][:3].tolist()}")


def same(a, b):
    """Equal values, NaN in the same places (fp16 inputs of a wide range hold infinities, which are kept as NaN)."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=0.0), torch.nan_to_num(b, nan=0.0))


def kept_oracle(x):
    """The checkpoint's values in 64 bits, by the definition."""
    cols = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    finite = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    top = finite.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # m in [1/2, 1)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    u = torch.where(torch.isinf(v), torch.full_like(v, math.nan), v) * torch.exp2(-e.double())
    step = torch.exp2((torch.frexp(u.abs())[1].clamp(min=-5) - 4).double())
    step = torch.where(torch.isfinite(u), step, torch.ones_like(step))
    out = torch.round(u / step) * step * torch.exp2(e.double())
    return out.flatten(-2)[..., :cols], (e + 127).squeeze(-1)


# ---------------------------------------------------------------------------------------------------------------------------
# Checkpoints
# ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (7, 33), (2, 40), (9, 128), (1, 4096), (301, 200), (4, 1001), (70001, 8)])
def test_checkpoint(dtype, rows, cols):
    from bioemu2_b200 import training as t

    x = (randn(gen(rows + cols), rows, cols) * torch.exp(3 * randn(gen(1), rows, 1))).to(dtype)
    kept = t.checkpoint8(x)
    want, exponents = kept_oracle(x)
    assert torch.equal(kept.exponents.long(), exponents.long())
    back = kept.restore()
    assert back.dtype == dtype and same(back, want.to(dtype))
    assert same(kept.restore(F32), want.float())


def test_checkpoint_of_special_values():
    from bioemu2_b200 import training as t

    big, small = torch.finfo(F32).max, 2.0 ** -149
    rows = [[0.0] * 32, [-0.0] * 32, [small, -small] * 16, [2.0 ** -126] * 32, [big, -big] + [1.0] * 30, [448.0, 449.0, 1.0, -464.0] * 8,
            [448.0, -448.0, 2.0 ** -9, 2.0 ** -10] * 8, [math.inf, -math.inf, 3.0, math.nan] * 8, [math.inf] * 32, [math.nan] * 32,
            [1.75, 1.7500001, 0.1, -0.3] * 8, [17.0, 18.0, 19.0, 240.0] * 8]
    for n in (32, 29):  # 29: a group that ends early, read value by value
        x = torch.tensor([r[:n] for r in rows], device=DEV)
        kept = t.checkpoint8(x)
        want, exponents = kept_oracle(x)
        assert torch.equal(kept.exponents.long(), exponents.long())
        assert torch.equal(torch.nan_to_num(kept.restore(), nan=-7.0), torch.nan_to_num(want.float(), nan=-7.0))


def test_checkpoint_of_strided_rows():
    from bioemu2_b200 import training as t

    base = randn(gen(5), 6, 5, 400)
    for view in (base[..., 8:136], base[..., 3:100], base[:, 1:4, :96], base.transpose(0, 1)[..., :64], base[..., ::2], base[:1].expand(4, 5, 400),
                 base[0, 0], base[:, 2, 7]):
        view = view if view.ndim > 1 or view.numel() > 6 else view[:, None]
        assert torch.equal(t.checkpoint8(view).restore(), kept_oracle(view)[0].float())


# ---------------------------------------------------------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------------------------------------------------------
def norm_oracle(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1 / torch.sqrt((d * d).mean(-1) + eps)
    n = d * rstd[..., None]
    return n * (1 if w is None else w.double()) + (0 if b is None else b.double()), mean, rstd, n


def check_norm(x, w, b, dy, eps=1e-5, out_dtype=None, keep=False, grad_dtype=None):
    from bioemu2_b200 import training as t

    out_dtype = out_dtype or x.dtype
    cols = x.shape[-1]
    y, mean, rstd, kept = t.layer_norm_forward(x, w, b, eps, out_dtype, keep)
    want, wmean, wrstd, n = norm_oracle(x, w, b, eps)
    sigma = 1 / wrstd
    wa = torch.ones(cols, device=DEV, dtype=torch.float64) if w is None else w.double().abs()
    ba = 0 if b is None else b.double().abs()
    assert y.dtype == out_dtype and (kept is None) == (not keep)
    check("y", y, want, 1.01 * half(out_dtype) * want.abs() + 64 * U * ((1 + n.abs()) * wa + ba) + tiny(out_dtype))
    check("mean", mean, wmean, U * (64 * sigma + 2 * wmean.abs()))
    check("rstd", rstd, wrstd, 64 * U * wrstd)
    if keep:
        assert torch.equal(kept.restore(F32), kept_oracle(x)[0].float())
    seen = kept_oracle(x)[0] if keep else x.double()
    dx, dw, db = t.layer_norm_backward(dy, kept if keep else x, mean, rstd, w, needs=(True, True, True), grad_dtype=grad_dtype)
    m, r = mean.double()[..., None], rstd.double()[..., None]
    n = (seen - m) * r
    dyd = dy.double()
    h = dyd * (1 if w is None else w.double())
    hn = h * n
    dxw = r * (h - h.mean(-1, keepdim=True) - n * hn.mean(-1, keepdim=True))
    size = r * (h.abs() + h.abs().mean(-1, keepdim=True) + n.abs() * hn.abs().mean(-1, keepdim=True))
    assert dx.dtype == x.dtype
    check("dx", dx, dxw, 1.01 * half(x.dtype) * dxw.abs() + 64 * U * size + tiny(x.dtype))
    gt = grad_dtype or (F32 if w is None else w.dtype)
    rows = x.numel() // cols
    depth = (64 + rows / 64) * U
    for name, got, terms in (("dw", dw, dyd * n), ("db", db, dyd)):
        terms = terms.reshape(-1, cols)
        s = terms.sum(0)
        assert got.dtype == gt
        check(name, got, s, 1.01 * half(gt) * s.abs() + depth * terms.abs().sum(0) + tiny(gt))
    return y, dx, dw, db


NORM_SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (17, 30), (9, 40), (33, 64), (130, 128), (7, 136), (19, 200), (257, 256), (65, 384), (12, 500), (3, 512),
              (6, 768), (11, 1000), (5, 1024), (4, 1027), (9, 2048), (3, 2056), (5, 4096), (2, 4100), (3, 8191), (4, 8192)]


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)], ids=str)
@pytest.mark.parametrize("keep", [False, True])
def test_layer_norm(rows, cols, types, keep):
    g = gen(cols)
    x = (randn(g, rows, cols) * 1.5 + 0.5).to(types[0])
    dy = randn(g, rows, cols).to(types[1])
    check_norm(x, 1 + 0.3 * randn(g, cols), 0.3 * randn(g, cols), dy, out_dtype=types[1], keep=keep)


@pytest.mark.parametrize("cols", [96, 101, 640, 3000])
@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(cols, w, b):
    g = gen(3)
    x, dy = randn(g, 21, cols), randn(g, 21, cols)
    check_norm(x, randn(g, cols) if w else None, randn(g, cols) if b else None, dy)


@pytest.mark.parametrize("param,grad", [(BF16, None), (F16, None), (F32, BF16), (BF16, F32)])
def test_layer_norm_parameter_types(param, grad):
    g = gen(4)
    x, dy = randn(g, 50, 128).bfloat16(), randn(g, 50, 128).bfloat16()
    check_norm(x, randn(g, 128).to(param), randn(g, 128).to(param), dy, grad_dtype=grad)


@pytest.mark.parametrize("rows,cols,dtype", [(262144 + 3, 16, BF16), (50000, 128, F32), (3001, 1536, F16), (1111, 4352, BF16), (40000, 200, F32)])
def test_layer_norm_many_rows(rows, cols, dtype):
    g = gen(6)
    x, dy = randn(g, rows, cols).to(dtype), randn(g, rows, cols).to(dtype)
    first = check_norm(x, randn(g, cols), randn(g, cols), dy)
    again = check_norm(x, torch.ones(cols, device=DEV), None, dy)
    assert torch.equal(first[3], again[3])  # db does not go by the weight: the same bits, run after run


def test_layer_norm_of_rows_far_from_zero():
    g = gen(7)
    for cols in (128, 384, 101, 3000):
        x = 1e4 + randn(g, 40, cols)
        check_norm(x, randn(g, cols), randn(g, cols), randn(g, 40, cols))


def test_layer_norm_of_constant_rows():
    from bioemu2_b200 import training as t

    x = torch.tensor([0.0, 5.0, -3e4], device=DEV)[:, None].expand(3, 384).contiguous()
    b = randn(gen(8), 384)
    y, mean, rstd, _ = t.layer_norm_forward(x, randn(gen(9), 384), b)
    assert torch.equal(y, b.expand(3, 384)) and torch.equal(mean, x[:, 0])
    assert torch.allclose(rstd, torch.full_like(rstd, 1e5 ** 0.5), rtol=4 * 2 ** -23)


def test_layer_norm_keeps_nan_and_infinity_to_their_rows():
    from bioemu2_b200 import training as t

    g = gen(10)
    for cols in (128, 77, 1000, 4096):
        x, dy, w = randn(g, 6, cols), randn(g, 6, cols), randn(g, cols)
        clean = t.layer_norm_forward(x, w)
        x2 = x.clone()
        x2[1, 3], x2[4, cols - 1] = math.nan, math.inf
        y, mean, rstd, _ = t.layer_norm_forward(x2, w)
        dx = t.layer_norm_backward(dy, x2, mean, rstd, w)[0]
        dx0 = t.layer_norm_backward(dy, x, clean[1], clean[2], w)[0]
        for r in range(6):
            if r in (1, 4):
                assert torch.isnan(y[r]).any() and torch.isnan(dx[r]).any()
            else:
                assert torch.equal(y[r], clean[0][r]) and torch.equal(dx[r], dx0[r])


def test_layer_norm_of_strided_rows():
    g = gen(11)
    base, grads = randn(g, 6, 5, 400), randn(g, 6, 5, 400)
    for cut in (lambda t: t[..., 8:136], lambda t: t[..., 3:100], lambda t: t[:, 1:4, :96], lambda t: t.transpose(0, 1)[..., :64],
                lambda t: t[..., ::2], lambda t: t[:1].expand(4, 5, 400), lambda t: t[0, 0]):
        x, dy = cut(base), cut(grads)
        check_norm(x, randn(g, x.shape[-1]), randn(g, x.shape[-1]), dy)


def test_views_that_negate():
    """The imaginary part of a conjugate is a view whose memory has the other sign."""
    from bioemu2_b200 import training as t

    x = torch.view_as_complex(randn(gen(18), 6, 64, 2)).conj().imag
    assert x.is_neg()
    assert torch.equal(t.layer_norm(x, x[0], x[1]), t.layer_norm(x.resolve_neg(), x[0].resolve_neg(), x[1].resolve_neg()))
    assert torch.equal(t.checkpoint8(x).restore(), t.checkpoint8(x.resolve_neg()).restore())


def test_layer_norm_without_rows():
    from bioemu2_b200 import training as t

    x = torch.empty(0, 7, 128, device=DEV)
    w = torch.ones(128, device=DEV)
    y, mean, rstd, kept = t.layer_norm_forward(x, w, w, checkpoint=True)
    assert y.shape == x.shape and mean.shape == (0, 7) and kept.restore().shape == x.shape
    dx, dw, db = t.layer_norm_backward(y, kept, mean, rstd, w)
    assert dx.shape == x.shape and not dw.any() and not db.any()


# ---------------------------------------------------------------------------------------------------------------------------
# Linear layer
# ---------------------------------------------------------------------------------------------------------------------------
def act_oracle(a, act):
    if act == "relu":
        return a.clamp(min=0)
    if act == "gelu":
        return 0.5 * a * torch.special.erfc(-a / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    return a * torch.sigmoid(a) if act == "silu" else a


def slope_oracle(a, act):
    with torch.enable_grad():
        a = a.detach().clone().requires_grad_()
        return torch.autograd.grad(act_oracle(a, act).sum(), a)[0].masked_fill((a == 0) & (act == "relu"), 0.0)


ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def check_linear(x, w, b, act, residual, dy, out_dtype=None, keep=False, save=True):
    from bioemu2_b200 import training as t

    k, n = x.shape[-1], w.shape[0]
    T = x.dtype
    out_dtype = out_dtype or (T if residual is None else residual.dtype)
    y, pre = t.linear_forward(x, w, b, act, residual, out_dtype, save=save)
    xd, wd = x.double().reshape(-1, k), w.double()
    a = xd @ wd.T + (0 if b is None else b.double())
    off = 2 * U * (k + 2) * (xd.abs() @ wd.abs().T) + (0 if b is None else 2 * U * b.double().abs())
    want = act_oracle(a, act) + (0 if residual is None else residual.double().reshape(-1, n))
    assert y.dtype == out_dtype and y.shape == x.shape[:-1] + (n,)
    bound = 1.2 * off + 16 * U * a.abs() + 1.01 * half(out_dtype) * want.abs() + tiny(out_dtype)
    check("y", y.reshape(-1, n), want, bound)
    if act is None:
        assert pre is None
    else:
        assert pre.dtype == (T if save is True else save)
        check("pre", pre.reshape(-1, n), a, off + 1.01 * half(pre.dtype) * a.abs() + tiny(pre.dtype))
    kept = t.checkpoint8(x) if keep else x
    dx, dw, db = t.linear_backward(dy, kept, w, pre, act)
    seen = kept_oracle(x)[0].reshape(-1, k).to(T).double() if keep else xd
    dyd = dy.double().reshape(-1, n)
    d = dyd if act is None else dyd * slope_oracle(pre.double().reshape(-1, n), act)
    wide = 16 * U * dyd.abs() * (0 if act is None else 1)
    off = wide + (0 if act is None and dy.dtype == T else 1.01 * half(T) * d.abs() + tiny(T))
    dxw = d @ wd
    assert dx.shape == x.shape and dx.dtype == T and dw.dtype == T and db.dtype == F32
    check("dx", dx.reshape(-1, k), dxw, off @ wd.abs() + 2 * U * n * (d.abs() @ wd.abs()) + 1.01 * half(T) * dxw.abs() + tiny(T))
    dww = d.T @ seen
    rows = xd.shape[0]
    check("dw", dw, dww, off.T @ seen.abs() + 2 * U * (rows + 8) * (d.abs().T @ seen.abs()) + 1.01 * half(T) * dww.abs() + tiny(T))
    dbw = d.sum(0)
    check("db", db, dbw, wide.sum(0) if act is None and not dyd.any() else (wide + (64 + rows / 64) * U * d.abs()).sum(0) + 2 * U * dbw.abs())
    return y, dx, dw, db


def linear_inputs(rows, k, n, dtype, seed=0):
    g = gen(seed + rows + k + n)
    x, w = randn(g, rows, k).to(dtype), (randn(g, n, k) / math.sqrt(k)).to(dtype)
    return g, x, w


LINEAR_SIZES = [(1, 8, 8), (1, 384, 1536), (2, 64, 64), (7, 72, 40), (31, 128, 512), (128, 64, 128), (129, 136, 264), (200, 512, 128), (74, 384, 1536),
                (300, 8, 1000), (300, 1000, 8), (515, 200, 328), (1000, 768, 384), (2049, 256, 320)]


@pytest.mark.parametrize("rows,k,n", LINEAR_SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ACTS, ids=str)
def test_linear(rows, k, n, dtype, act):
    g, x, w = linear_inputs(rows, k, n, dtype)
    check_linear(x, w, randn(g, n), act, None, randn(g, rows, n).to(dtype))


@pytest.mark.parametrize("rows,k,n", [(5, 128, 64), (130, 72, 200), (700, 384, 128), (257, 512, 520)])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("act,bias,keep", [(None, True, False), (None, False, True), ("silu", False, True), ("gelu", True, False)])
def test_linear_with_residual(rows, k, n, dtype, out, act, bias, keep):
    g, x, w = linear_inputs(rows, k, n, dtype)
    check_linear(x, w, randn(g, n) if bias else None, act, 3 * randn(g, rows, n).to(out), randn(g, rows, n).to(out), keep=keep)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_to_fp32(dtype):
    g, x, w = linear_inputs(333, 96, 160, dtype)
    check_linear(x, w, randn(g, 160), "gelu", None, randn(g, 333, 160), out_dtype=F32)


@pytest.mark.parametrize("rows,k,n", [(3, 64, 24), (200, 96, 160), (129, 264, 72), (3000, 128, 512)])
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_saving_fp32(rows, k, n, out, residual):
    g, x, w = linear_inputs(rows, k, n, BF16)
    check_linear(x, w, randn(g, n), "gelu", randn(g, rows, n).to(out) if residual else None, randn(g, rows, n).to(out), out_dtype=out, save=F32)


@pytest.mark.parametrize("rows,k,n,act", [(41209, 128, 512, "silu"), (41209, 512, 128, None), (70003, 64, 256, "gelu"), (20011, 768, 768, None)])
def test_linear_many_rows(rows, k, n, act):
    g, x, w = linear_inputs(rows, k, n, BF16)
    dy = (randn(g, rows, n) / math.sqrt(rows)).bfloat16()
    one = check_linear(x, w, randn(g, n), act, None, dy, keep=rows == 70003)
    if rows == 20011:  # and its 8-bit form, in two parts of the contraction and more
        check_linear(x, w, None, act, None, dy, keep=True)
        check_linear(x[:700], w, None, act, None, dy[:700], keep=True)
    two = check_linear(x, w, randn(gen(1), n), None, None, dy)
    if act is None:
        assert torch.equal(one[1], two[1]) and torch.equal(one[2], two[2])  # the same bits, run after run


@pytest.mark.parametrize("rows,k,n", [(1025, 64, 8), (1100, 128, 256), (1200, 32, 384), (9500, 8, 64), (9600, 72, 120), (50000, 136, 128), (12345, 56, 72), (90001, 256, 104), (40000, 200, 200),
                                      (30001, 128, 136), (85000, 256, 256), (15000, 64, 296), (83001, 128, 384), (40111, 104, 392), (19000, 128, 512),
                                      (9555, 40, 504), (100003, 120, 488)])
@pytest.mark.parametrize("act,dtype,out,keep", [("silu", BF16, BF16, False), ("gelu", F16, F16, True), (None, BF16, F32, True), ("gelu_tanh", BF16, F32, False),
                                                (None, F16, F16, False), ("relu", BF16, BF16, True)])
def test_linear_with_more_rows_than_columns(rows, k, n, act, dtype, out, keep):
    """Sizes whose backward pass is one kernel, or just is not: one to four pieces of n, one or two of k, the last of each cut short."""
    g, x, w = linear_inputs(rows, k, n, dtype)
    dy = (randn(g, rows, n) / math.sqrt(rows)).to(out)
    one = check_linear(x, w, randn(g, n), act, None, dy, out_dtype=out, keep=keep)
    from bioemu2_b200 import training as t

    y, pre = t.linear_forward(x, w, randn(gen(2), n), act, save=True)
    a = t.linear_backward(dy, x, w, pre, act)
    assert all(torch.equal(u, v) for u, v in zip(a, t.linear_backward(dy, x, w, pre, act)))
    assert not torch.isnan(one[1]).any()


def test_linear_of_strided_operands():
    g = gen(12)
    base, grads, wide = randn(g, 6, 5, 400).bfloat16(), randn(g, 6, 5, 800).bfloat16(), (0.1 * randn(g, 300, 600)).bfloat16()
    for cut in (lambda t: t[..., 8:136], lambda t: t[..., 3:99], lambda t: t[:, 1:4, :96], lambda t: t.transpose(0, 1)[..., :64],
                lambda t: t[..., ::2], lambda t: t[:1].expand(4, 5, 400), lambda t: t[0, 0]):
        x = cut(base)
        k = x.shape[-1]
        for w in (wide[:72, :k], wide[3:67, 5:5 + k], wide.T[:72, :k] if k <= 300 else wide[:72, :k]):
            dy = grads[: x.shape[0], : x.shape[1], 8:8 + w.shape[0]] if x.ndim == 3 and x.shape[0] <= 6 and x.shape[1] <= 5 else \
                randn(g, *x.shape[:-1], w.shape[0]).bfloat16()
            check_linear(x, w, None, "silu", None, dy)


def test_linear_bounds_of_the_output_are_kept():
    """Rows and columns behind the last one of a tile stay as they were: outputs are views into larger buffers at the C entry."""
    from bioemu2_b200 import _lib

    g, x, w = linear_inputs(37, 72, 40, BF16)
    out = torch.full((64, 40), 7.0, device=DEV, dtype=BF16)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.lib.b200_linear_act_fwd(x.data_ptr(), 72, w.data_ptr(), 72, None, 0, None, 40, out.data_ptr(), None, 37, 72, 40, 0, 0, 0, stream))
    assert (out[37:] == 7).all()
    check("y", out[:37], x.double() @ w.double().T, 1.0 * half(BF16) * 1.01 * (x.double() @ w.double().T).abs() + 2 * U * 80 * (x.double().abs() @ w.double().abs().T))


def test_refusals_of_the_c_entries():
    """Arguments that only another host can get wrong: the library says so and launches nothing."""
    import ctypes

    from bioemu2_b200 import _lib

    x = randn(gen(19), 16, 64)
    xb = x.bfloat16()
    y, f, i = torch.empty_like(x), torch.empty(16, device=DEV), torch.empty(16, 64, device=DEV, dtype=torch.uint8)
    st = torch.cuda.current_stream().cuda_stream
    p, lib = (lambda v: v.data_ptr()), _lib.lib
    before = _lib.launch_count()

    def refused(status, code=_lib.ERR_INVALID_ARGUMENT):
        assert status == code and _lib.last_error()

    norm = [p(x), 64, None, None, p(y), p(f), p(f), None, None, 16, 64, 1e-5, 1, 1, st]
    for at, value in ((0, None), (1, 63), (4, None), (5, None), (7, p(i)), (9, -1), (10, 0), (10, 8193), (12, 3), (13, 7), (0, p(x) + 2), (12, 0)):
        refused(lib.b200_layer_norm_save_fwd(*[value if j == at else v for j, v in enumerate(norm)]))
    size = lib.b200_layer_norm_bwd_workspace_bytes(16, 64)
    ws = torch.empty(size, device=DEV, dtype=torch.uint8)
    grad = [p(x), 64, p(x), 64, None, None, p(f), p(f), None, p(y), p(f), p(f), 16, 64, 1, 1, 1, p(ws), size, st]
    for at, value in ((0, None), (2, None), (6, None), (1, 8), (3, 8), (4, p(i)), (13, 0), (16, 9), (14, 0)):
        refused(lib.b200_layer_norm_bwd(*[value if j == at else v for j, v in enumerate(grad)]))
    refused(lib.b200_layer_norm_bwd(*grad[:18], size - 1, st), _lib.ERR_WORKSPACE)
    refused(lib.b200_layer_norm_bwd(*grad[:17], None, size, st), _lib.ERR_WORKSPACE)
    assert lib.b200_layer_norm_bwd_workspace_bytes(0, 64) == 0 and lib.b200_layer_norm_bwd_workspace_bytes(16, 9000) == 0
    keep = [p(x), 64, p(i), p(i), 16, 64, 1, st]
    for at, value in ((0, None), (2, None), (3, None), (1, 63), (4, -1), (5, 0), (6, 3)):
        refused(lib.b200_checkpoint8_fwd(*[value if j == at else v for j, v in enumerate(keep)]))
    refused(lib.b200_checkpoint8_restore(p(i), None, p(y), 16, 64, 1, st))
    refused(lib.b200_checkpoint8_restore(p(i), p(i), p(y), 16, 64, 5, st))
    fwd = [p(xb), 64, p(xb), 64, None, 0, None, 16, p(y), None, 16, 64, 16, 0, 0, 0, st]
    for at, value in ((0, None), (2, None), (8, None), (1, 32), (1, 68), (3, 60), (5, 5), (5, -1), (10, -1), (11, 60), (12, 12), (13, 1), (14, 2), (0, p(xb) + 2),
                      (8, p(y) + 8)):
        refused(lib.b200_linear_act_fwd(*[value if j == at else v for j, v in enumerate(fwd)]))
    refused(lib.b200_linear_act_fwd(*[p(y) if j == 9 else 2 if j == 15 else v for j, v in enumerate(fwd)]))
    good = dict(dy=p(xb), dy_pitch=16, x=p(xb), x_pitch=64, w=p(xb), w_pitch=64, pre=p(xb), pre_pitch=16, dx=p(y), dw=p(y), db=p(f), rows=16, k=64, n=16, act=2,
                dtype=0, dy_dtype=0, pre_dtype=0, db_dtype=1)
    for wrong in (dict(dy=None), dict(x=None), dict(w=None), dict(pre=None), dict(values=p(i)), dict(dy_pitch=8), dict(x_pitch=56), dict(w_pitch=70), dict(pre_pitch=20),
                  dict(rows=-1), dict(k=63), dict(n=0), dict(act=9), dict(dtype=1), dict(dy_dtype=2), dict(pre_dtype=2), dict(db_dtype=4), dict(dx=p(y) + 4)):
        g = _lib.LinearGrad(**{**good, **wrong})
        refused(lib.b200_linear_act_bwd(ctypes.byref(g), p(ws), 1 << 30, st))
    g = _lib.LinearGrad(**good)
    need = lib.b200_linear_act_bwd_workspace_bytes(ctypes.byref(g))
    assert need > 0
    refused(lib.b200_linear_act_bwd(ctypes.byref(g), p(ws), need - 1, st), _lib.ERR_WORKSPACE)
    refused(lib.b200_linear_act_bwd(ctypes.byref(g), None, need, st), _lib.ERR_WORKSPACE)
    refused(lib.b200_linear_act_bwd(None, p(ws), need, st))
    assert _lib.launch_count() == before


def test_linear_without_rows():
    from bioemu2_b200 import training as t

    x, w = torch.empty(0, 3, 64, device=DEV, dtype=BF16), torch.ones(128, 64, device=DEV, dtype=BF16)
    y, pre = t.linear_forward(x, w, None, "gelu", save=True)
    dx, dw, db = t.linear_backward(y, x, w, pre, "gelu")
    assert y.shape == (0, 3, 128) and dx.shape == x.shape and dw.shape == w.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("rows", [40, 1200])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_far_out(rows, act):
    """Values before the activation of any size, infinities among them: the activation is the value or nothing, its slope one or
    nothing, and a NaN stays with its element (neighbours share a reciprocal).  1200 rows: the backward pass in one kernel."""
    from bioemu2_b200 import training as t

    sizes = [6.0, 9.0, 12.0, 30.0, 41.0, 42.0, 64.0, 100.0, 1e4, 1e10, 1e19, 1e20, 1e30, 3e38, math.inf]
    a = torch.tensor([s * v for v in sizes for s in (-1, 1)] + [math.nan, 0.5], device=DEV).bfloat16()[None].expand(rows, 32)
    x = torch.zeros(rows, 8, device=DEV, dtype=BF16)
    w = torch.zeros(32, 8, device=DEV, dtype=BF16)
    bias = a[0].float()
    y, pre = t.linear_forward(x, w, bias, act, out_dtype=F32, save=True)
    assert torch.equal(torch.nan_to_num(pre, 7.0), torch.nan_to_num(a, 7.0))
    want = torch.where(a[0].double() > 0, a[0].double(), torch.zeros(32, device=DEV, dtype=torch.float64))
    small = a[0].double().abs() < 50  # here the formula itself: silu of 12 is 12 less 7e-5
    want = torch.where(small, act_oracle(a[0].double(), act), want)
    assert torch.isnan(y[:, 30]).all()
    fine = [i for i in range(32) if i != 30]
    got = y.double()[:, fine]
    same_inf = torch.isinf(got) & (got == want[fine])
    # what is nothing may be 41.5 x 2^-60: the sigmoid's exponent ends at 60, and the value that multiplies it at 41.5 = 60 ln 2
    bound = 16 * U * want[fine].abs() + 16 * U * 10 * small[fine] + 1e-7 * (a[0, fine].double().abs() < 50) + 42 * 2.0 ** -60
    assert (same_inf | ((got - want[fine]).abs() <= bound)).all()
    dy = torch.ones(rows, 32, device=DEV)
    dx, dw, db = t.linear_backward(dy, x, w, pre, act)
    slope = torch.where(a[0].double() > 0, 1.0, 0.0)
    slope = torch.where(small, slope_oracle(a[0].double(), act), slope)
    off = (db.double()[fine] / rows - slope[fine]).abs()
    assert torch.isnan(db[30]) and (off <= 32 * U * (1 + a[0, fine].double().abs().clamp(max=50))).all(), off


def test_linear_passes_what_is_not_finite():
    from bioemu2_b200 import training as t

    g, x, w = linear_inputs(40, 64, 72, F16)
    x[3, 5], x[17, 0] = math.nan, math.inf
    y, pre = t.linear_forward(x, w, None, "relu", save=True)
    rows = torch.arange(40, device=DEV)
    fine = (rows != 3) & (rows != 17)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[fine]).all()
    assert torch.isnan(t.linear_backward(randn(g, 40, 72).half(), x, w, pre, "relu")[0][3]).all()


# ---------------------------------------------------------------------------------------------------------------------------
# As they are used
# ---------------------------------------------------------------------------------------------------------------------------
def transition(t, d, hidden, act, checkpoint, dtype):
    torch.manual_seed(0)
    norm = t.LayerNorm(d, out_dtype=dtype, checkpoint=checkpoint, device=DEV)
    up = t.Linear(d, hidden, activation=act, checkpoint=checkpoint, device=DEV)
    down = t.Linear(hidden, d, bias=False, checkpoint=checkpoint, device=DEV)
    with torch.no_grad():
        norm.weight.add_(0.2 * torch.randn_like(norm.weight))
        norm.bias.add_(0.2 * torch.randn_like(norm.bias))
    return norm, up, down


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("d,hidden,act", [(128, 512, "silu"), (384, 1536, "gelu")])
def test_residual_transition(d, hidden, act, checkpoint):
    """LN, widening layer, narrowing layer with the fp32 stream as its residual: value and gradients against 64 bits.  Every step
    rounds its operands to bf16, so the bound is on the norm of the difference: three roundings on the way to y's update, five
    on the way to the first gradients, each 2^-9 at most of the norm it meets, and the 8-bit form's 2^-4 where it is used."""
    from bioemu2_b200 import training as t

    norm, up, down = transition(t, d, hidden, act, checkpoint, BF16)
    g = gen(13)
    z = randn(g, 2, 19, 17, d).requires_grad_()
    dz = randn(g, 2, 19, 17, d)
    out = down(up(norm(z)), residual=z)
    out.backward(dz)
    params = [norm.weight, norm.bias, up.weight, up.bias, down.weight]
    got = [z.grad] + [p.grad for p in params]
    z64 = z.detach().double().requires_grad_()
    p64 = [p.detach().double().requires_grad_() for p in params]
    a = torch.nn.functional.layer_norm(z64, (d,), p64[0], p64[1]) @ p64[2].T + p64[3]
    want = act_oracle(a, act) @ p64[4].T + z64
    want.backward(dz.double())
    assert out.dtype == F32
    update = want - z64
    assert float((out.detach().double() - want.detach()).norm() / update.detach().norm()) < 5 * 2 ** -8
    for name, a, b in zip(["z", "norm.weight", "norm.bias", "up.weight", "up.bias", "down.weight"], got, [z64.grad] + [p.grad for p in p64]):
        assert a.dtype == F32 and a.shape == b.shape, name
        assert float((a.double() - b).norm() / b.norm()) < 8 * 2 ** -8 + (2 ** -4 if checkpoint else 0), name


def test_gradients_against_differences():
    """Directional derivatives of the functions themselves, in fp32 outputs, against what backward says."""
    from bioemu2_b200 import training as t

    g = gen(14)
    x, w, b, u = randn(g, 33, 96), 1 + 0.2 * randn(g, 96), randn(g, 96), randn(g, 33, 96)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    (t.layer_norm(*leaves) * u).sum().backward()
    for i, v in enumerate((x, w, b)):
        step = randn(g, *v.shape)
        h = 2.0 ** -6
        vals = []
        for s in (h, -h):
            args = [x, w, b]
            args[i] = v + s * step
            vals.append((t.layer_norm(*args).double() * u.double()).sum())
        difference = (vals[0] - vals[1]) / (2 * h)
        said = (leaves[i].grad.double() * step.double()).sum()
        # h^2 / 6 of the third derivative, which is of the size of the terms, and the differences' rounding U / h of the sum
        size = float((leaves[i].grad.double() * step.double()).abs().sum())
        assert abs(float(difference - said)) < 4 * h * h * size + 64 * U / h * float(u.abs().sum())


def test_functions_return_what_the_passes_do_and_only_what_is_wanted():
    from bioemu2_b200 import training as t

    g = gen(15)
    x = randn(g, 40, 64).bfloat16()
    w, b = (0.2 * randn(g, 48, 64)).bfloat16(), randn(g, 48)
    r, dy = randn(g, 40, 48).bfloat16(), randn(g, 40, 48).bfloat16()
    y, pre = t.linear_forward(x, w, b, "silu", r, save=True)
    want = dict(zip("xwb", t.linear_backward(dy, x, w, pre, "silu")))
    want["r"] = dy
    for wanted in itertools.chain.from_iterable(itertools.combinations("xwbr", n) for n in range(5)):
        args = {k: v.clone().requires_grad_(k in wanted) for k, v in dict(x=x, w=w, b=b, r=r).items()}
        out = t.linear(args["x"], args["w"], args["b"], "silu", args["r"])
        assert torch.equal(out, y) and out.requires_grad == bool(wanted)
        if wanted:
            out.backward(dy)
        for k, v in args.items():
            assert (v.grad is not None) == (k in wanted)
            if v.grad is not None:
                assert torch.equal(v.grad, want[k]), k
    xn, wn, bn, dyn = randn(g, 40, 64), randn(g, 64), randn(g, 64), randn(g, 40, 64)
    y, mean, rstd, _ = t.layer_norm_forward(xn, wn, bn)
    want = dict(zip("xwb", t.layer_norm_backward(dyn, xn, mean, rstd, wn)))
    for wanted in itertools.chain.from_iterable(itertools.combinations("xwb", n) for n in range(4)):
        args = {k: v.clone().requires_grad_(k in wanted) for k, v in dict(x=xn, w=wn, b=bn).items()}
        out = t.layer_norm(args["x"], args["w"], args["b"])
        assert torch.equal(out, y) and out.requires_grad == bool(wanted)
        if wanted:
            out.backward(dyn)
        for k, v in args.items():
            assert (v.grad is not None) == (k in wanted)
            if v.grad is not None:
                assert torch.equal(v.grad, want[k]), k


def test_gradient_of_expanded_and_strided_upstream():
    """dy as autograd hands it over after a sum (expanded, all strides zero) and after a transpose."""
    from bioemu2_b200 import training as t

    g = gen(16)
    w = randn(g, 128)
    for reduce in (lambda y: y.float().sum(), lambda y: (y.float().transpose(0, 1) * torch.arange(1.0, 6.0, device=DEV)[:, None, None]).sum()):
        x = randn(g, 4, 5, 128).requires_grad_()
        reduce(t.layer_norm(x, w)).backward()
        xd = x.detach().double().requires_grad_()
        reduce64 = reduce(torch.nn.functional.layer_norm(xd, (128,), w.double()).double())
        reduce64.backward()
        assert float((x.grad.double() - xd.grad).norm()) <= 1e-6 * float(xd.grad.norm()) + 1e-5
        xl, wl = randn(g, 4, 5, 128).bfloat16().requires_grad_(), (0.1 * randn(g, 64, 128)).bfloat16()
        reduce(t.linear(xl, wl)).backward()
        scale = torch.arange(1.0, 6.0, device=DEV).double() if xl.grad[0, 0].ne(xl.grad[0, 1]).any() else torch.ones(5, device=DEV).double()
        want = scale[None, :, None] * wl.double().sum(0)
        assert float((xl.grad.double() - want).abs().max()) <= 2 ** -8 * float(want.abs().max())


def test_on_another_stream_and_captured():
    """A side stream, two graphs of the same call replayed at the same time on two streams, and new inputs on replay."""
    from bioemu2_b200 import training as t

    g = gen(17)
    rows, k, n = 1000, 128, 256
    w, b = (0.1 * randn(g, n, k)).bfloat16(), randn(g, n)
    gamma = randn(g, k)

    def step(z, dy):
        x, mean, rstd, kept = t.layer_norm_forward(z, gamma, None, out_dtype=BF16, checkpoint=True)
        y, pre = t.linear_forward(x, w, b, "gelu", save=True)
        dx, dw, db = t.linear_backward(dy, t.checkpoint8(x), w, pre, "gelu")
        return (y, dw, db) + t.layer_norm_backward(dx, kept, mean, rstd, gamma)

    data = [(randn(g, rows, k), randn(g, rows, n).bfloat16()) for _ in range(4)]
    want = [step(*d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*data[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for i in range(2):
        z, dy = data[i][0].clone(), data[i][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(z, dy)
        graphs.append((graph, z, dy, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for turn in (0, 2):
        for i, (graph, z, dy, out, stream) in enumerate(graphs):
            z.copy_(data[turn + i][0])
            dy.copy_(data[turn + i][1])
        torch.cuda.synchronize()
        for graph, _, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, _, out, _) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[turn + i]))
