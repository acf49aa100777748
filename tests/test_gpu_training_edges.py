"""Edges of the training operators: calls and values that their other tests leave out."""
import math

import pytest
import torch

from test_gpu_training_operators import BF16, DEV, F16, F32, U, check, check_linear, gen, half, kept_oracle, linear_inputs, randn, slope_oracle, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,n,act", [(256, 128, "silu"), (200, 256, "gelu"), (128, 384, None), (128, 512, "silu"), (72, 264, "relu")])
@pytest.mark.parametrize("tiles", [148, 149, 222, 223, 300])
def test_paired_backward_ends_after_any_number_of_tiles(k, n, act, tiles):
    """Two CTAs share a layer's k, and each waits at its end for the other's last arrivals at the slots that were used: slots used
    once, twice, an even and an odd number of times, and not at all.  A wait for a phase that never comes would be in the status."""
    from bioemu2_b200 import training as t

    rows = tiles * 128 - 5
    g, x, w = linear_inputs(rows, k, n, BF16)
    dy = (randn(g, rows, n) / math.sqrt(rows)).bfloat16()
    check_linear(x, w, randn(g, n), act, None, dy)
    pre = None if act is None else randn(g, rows, n).bfloat16()
    first = t.linear_backward(dy, x, w, pre, act)
    for _ in range(20):  # one launch behind the other: what one leaves on its way would land in the next one's
        last = t.linear_backward(dy, x, w, pre, act)
    check("status", first[2], first[2].double(), torch.zeros_like(first[2], dtype=torch.float64))
    assert all(torch.equal(a, b) for a, b in zip(first, last))


def largest_values(dtype):
    """Magnitudes whose rounding to e4m3 has no place in the type: the last 1/32 of its last binade, and what lies around it."""
    big = torch.finfo(dtype).max
    step = big * torch.finfo(dtype).eps / 2  # at the top of the last binade
    last = 2.0 ** math.floor(math.log2(big))
    return [big, big - step, 1.9375 * last, 1.9375 * last - step, 1.9375 * last + step, 1.875 * last, 1.75 * last, 1.75 * last + step, last]


def kept_finite(x):
    """What a checkpoint gives back in x's type: its values, finite ones no larger than the type's."""
    big = torch.finfo(x.dtype).max
    return kept_oracle(x)[0].clamp(-big, big)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [32, 29, 96])
def test_checkpoint_of_the_largest_finite_values(dtype, cols):
    from bioemu2_b200 import training as t

    tops = torch.tensor(largest_values(dtype), device=DEV, dtype=torch.float64).to(dtype)
    assert torch.isfinite(tops).all()
    x = torch.cat([tops, -tops])[:, None] * torch.tensor([1.0, -0.5, 2.0 ** -6, 0.0], device=DEV, dtype=dtype).repeat(24)[:cols]
    back = t.checkpoint8(x).restore()
    assert torch.isfinite(back).all() and torch.equal(back, kept_finite(x).to(dtype))
    assert ((back.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * x.double().abs().amax(-1, keepdim=True)).all()
    x[3, 1], x[4, 2], x[5, 0] = math.inf, -math.inf, math.nan  # which are not finite, and stay marked
    back = t.checkpoint8(x).restore()
    assert torch.equal(torch.isnan(back), ~torch.isfinite(x)) and not torch.isinf(back).any()
    assert torch.equal(back.nan_to_num(nan=7.0), kept_finite(x).to(dtype).nan_to_num(nan=7.0))


def test_checkpoint_restored_in_a_shorter_type():
    from bioemu2_b200 import training as t

    x = torch.tensor([[1e6, -7e4, 6e4, 1.0] * 8, [3e38, -3.4e38, 1e38, 0.0] * 8, [math.inf, math.nan, 1e6, -1e6] * 8], device=DEV)
    want = kept_oracle(x)[0]
    for dtype in (F16, BF16, F32):
        big = torch.finfo(dtype).max
        back = t.checkpoint8(x).restore(dtype)
        assert torch.equal(torch.isnan(back), torch.isnan(want))
        assert torch.equal(back.nan_to_num(nan=7.0), want.clamp(-big, big).to(dtype).nan_to_num(nan=7.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [128, 101, 1024, 3001])
def test_layer_norm_gradients_from_a_checkpoint_of_the_largest_values(dtype, cols):
    """Finite rows give finite gradients: those of the values that restore() gives."""
    from bioemu2_b200 import training as t

    g = gen(31)
    x, dy = randn(g, 12, cols).to(dtype), randn(g, 12, cols).to(dtype)
    tops = torch.tensor(largest_values(dtype), device=DEV, dtype=torch.float64).to(dtype)
    x[torch.arange(9), torch.arange(9) * 11] = tops
    w = randn(g, cols)
    _, mean, rstd, kept = t.layer_norm_forward(x, w, checkpoint=True)
    got = t.layer_norm_backward(dy, kept, mean, rstd, w)
    n = (kept_finite(x) - mean.double()[:, None]) * rstd.double()[:, None]
    h = dy.double() * w.double()
    hn = h * n
    r = rstd.double()[:, None]
    dx = r * (h - h.mean(-1, keepdim=True) - n * hn.mean(-1, keepdim=True))
    size = r * (h.abs() + h.abs().mean(-1, keepdim=True) + n.abs() * hn.abs().mean(-1, keepdim=True))
    check("dx", got[0], dx, 1.01 * half(dtype) * dx.abs() + 64 * U * size + tiny(dtype))
    dw = dy.double() * n
    check("dw", got[1], dw.sum(0), 65 * U * dw.abs().sum(0) + tiny(F32))


@pytest.mark.parametrize("rows,k,n,act", [(300, 200, 328, None), (3000, 768, 768, None), (1200, 64, 64, None), (1100, 128, 256, "relu"), (148 * 128, 128, 512, "relu"),
                                          (40, 64, 72, "relu")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_gradient_from_a_checkpoint_of_the_largest_values(rows, k, n, act, dtype):
    """dw of finite activations is finite, whichever kernel makes it; a column of dy of zeros gives zeros."""
    from bioemu2_b200 import training as t

    g, x, w = linear_inputs(rows, k, n, dtype)
    tops = torch.tensor(largest_values(dtype), device=DEV, dtype=torch.float64).to(dtype)
    x[torch.arange(9) * 4, torch.arange(9) * 7] = tops
    x[rows - 1, k - 1] = -torch.finfo(dtype).max
    dy = (1e-3 * randn(g, rows, n)).to(dtype)
    dy[:, 3] = 0
    pre = None if act is None else torch.ones(rows, n, device=DEV, dtype=dtype)
    dw = t.linear_backward(dy, t.checkpoint8(x), w, pre, act)[1]
    seen, d = kept_finite(x), dy.double()
    want = d.T @ seen
    # 2 U a term for the products' sum, a rounding for the output
    check("dw", dw, want, 2 * U * (rows + 8) * (d.abs().T @ seen.abs()) + 1.01 * half(dtype) * want.abs() + tiny(dtype))
    assert not dw[3].any()


class Wrapper(torch.Tensor):
    """A tensor around another one, with its shape, type and device and no memory."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} of a wrapper")


def freed(t):
    t = t.clone()
    t.untyped_storage().resize_(0)
    return t


@pytest.mark.parametrize("wrap", [Wrapper, freed])
def test_tensors_without_memory_are_refused(wrap):
    """Their null pointers would stand for arguments that were not given: a weight of one, a bias or a residual of zero."""
    from bioemu2_b200 import _lib, training as t

    g = gen(34)
    x, dy, mean, w, b = randn(g, 6, 64), randn(g, 6, 64), randn(g, 6), randn(g, 64), randn(g, 64)
    kept = t.checkpoint8(x)
    xl, wl, bl, r, pre = randn(g, 6, 64).bfloat16(), randn(g, 48, 64).bfloat16(), randn(g, 48), randn(g, 6, 48).bfloat16(), randn(g, 6, 48)
    before = _lib.launch_count()
    for call in (lambda: t.layer_norm(wrap(x)), lambda: t.layer_norm(x, wrap(w), b), lambda: t.layer_norm(x, w, wrap(b)),
                 lambda: t.layer_norm(x, wrap(w).requires_grad_(), b), lambda: t.checkpoint8(wrap(x)),
                 lambda: t.Checkpoint8(wrap(kept.values), kept.exponents, F32).restore(), lambda: t.Checkpoint8(kept.values, wrap(kept.exponents), F32).restore(),
                 lambda: t.layer_norm_backward(wrap(dy), x, mean, mean), lambda: t.layer_norm_backward(dy, wrap(x), mean, mean),
                 lambda: t.layer_norm_backward(dy, x, wrap(mean), mean), lambda: t.layer_norm_backward(dy, x, mean, wrap(mean)),
                 lambda: t.layer_norm_backward(dy, x, mean, mean, wrap(w)), lambda: t.linear(wrap(xl), wl), lambda: t.linear(xl, wrap(wl)),
                 lambda: t.linear(xl, wl, wrap(bl)), lambda: t.linear(xl, wl, bl, "silu", wrap(r)), lambda: t.linear(xl, wl, wrap(bl).requires_grad_()),
                 lambda: t.linear_backward(wrap(r), xl, wl), lambda: t.linear_backward(r, wrap(xl), wl), lambda: t.linear_backward(r, xl, wrap(wl)),
                 lambda: t.linear_backward(r, xl, wl, wrap(pre), "silu")):
        with pytest.raises(ValueError, match="memory of its own"):
            call()
    assert _lib.launch_count() == before


@pytest.mark.parametrize("wt,bt", [(BF16, F32), (F16, F32), (F32, BF16), (F32, F16), (BF16, F16), (F16, BF16)], ids=str)
def test_layer_norm_parameters_of_two_types(wt, bt):
    """Each parameter's gradient is the fp32 sum rounded once, to that parameter's type."""
    from bioemu2_b200 import training as t

    g = gen(32)
    x, dy = randn(g, 900, 64).bfloat16(), (40 * randn(g, 900, 64) + 90).bfloat16()  # sums of 81000: beyond fp16's largest value
    w, b = randn(g, 64).to(wt).requires_grad_(), randn(g, 64).to(bt).requires_grad_()
    t.layer_norm(x, w, b).backward(dy)
    assert w.grad.dtype == wt and b.grad.dtype == bt
    want = dy.double().sum(0)
    mean, rstd = (v.double()[:, None] for v in t.layer_norm_forward(x)[1:3])
    terms = dy.double() * (x.double() - mean) * rstd
    for grad, sums, size in ((b.grad, want, dy.double().abs().sum(0)), (w.grad, terms.sum(0), terms.abs().sum(0))):
        if grad.dtype == F16 and float(sums.abs().max()) > 65504:
            assert torch.isinf(grad).any()
            continue
        check("gradient", grad, sums, (64 + 900 / 64) * U * size + 1.01 * half(grad.dtype) * sums.abs() + tiny(grad.dtype))


def test_statistics_as_views_that_negate():
    from bioemu2_b200 import training as t

    g = gen(33)
    x, dy, w = randn(g, 6, 64), randn(g, 6, 64), randn(g, 64)
    _, mean, rstd, _ = t.layer_norm_forward(x, w)
    want = t.layer_norm_backward(dy, x, mean, rstd, w)
    zero = torch.zeros(6, device=DEV)
    views = [torch.complex(zero, -v).conj().imag for v in (mean, rstd)]
    assert all(v.is_neg() and torch.equal(v, u) for v, u in zip(views, (mean, rstd)))
    flat = [torch.view_as_complex(torch.stack([zero, -v], -1))[:1].conj().imag for v in (mean, rstd)]  # one element: contiguous as it lies
    assert all(torch.equal(a, b) for a, b in zip(t.layer_norm_backward(dy, x, *views, w), want))
    assert all(v.is_neg() and v.is_contiguous() for v in flat)
    one = t.layer_norm_backward(dy[:1], x[:1], mean[:1], rstd[:1], w)
    assert all(torch.equal(a, b) for a, b in zip(t.layer_norm_backward(dy[:1], x[:1], *flat, w), one))
    


def large(g, *shape):
    return torch.empty(*shape, device=DEV, dtype=BF16).normal_(generator=g)


def test_checkpoint_of_the_widest_row():
    """One row of 2^31 - 1 columns, whose groups are counted to the last, shorter one."""
    from bioemu2_b200 import training as t

    x = large(gen(41), 2 ** 31 - 1)
    kept = t.checkpoint8(x)
    assert kept.exponents.numel() == 2 ** 26
    back = kept.restore()
    for at in (0, 2 ** 30, 2 ** 31 - 4096):
        part = x[at:at + 4096]
        assert torch.equal(back[at:at + 4096], kept_oracle(part)[0].bfloat16())
        assert torch.equal(kept.exponents[at // 32:at // 32 + 128].long(), kept_oracle(part)[1].long())


def test_layer_norm_of_more_elements_than_32_bits_count():
    from bioemu2_b200 import training as t

    rows, cols = 2 ** 24 + 3001, 128
    g = gen(42)
    x, dy, w, b = large(g, rows, cols), large(g, rows, cols), randn(g, cols), randn(g, cols)
    y, mean, rstd, kept = t.layer_norm_forward(x, w, b, checkpoint=True)
    end = slice(rows - 5000, rows)
    want = t.layer_norm_forward(x[end], w, b, checkpoint=True)
    assert torch.equal(y[end], want[0]) and torch.equal(mean[end], want[1]) and torch.equal(rstd[end], want[2])
    assert torch.equal(kept.values[end].view(torch.uint8), want[3].values.view(torch.uint8)) and torch.equal(kept.exponents[end], want[3].exponents)
    dx = t.layer_norm_backward(dy, kept, mean, rstd, w)[0]
    assert torch.equal(dx[end], t.layer_norm_backward(dy[end], want[3], mean[end], rstd[end], w)[0])
    del kept
    dx = t.layer_norm_backward(dy, x, mean, rstd, w)[0]
    assert torch.equal(dx[end], t.layer_norm_backward(dy[end], x[end], mean[end], rstd[end], w)[0])


@pytest.mark.parametrize("k,n", [(128, 128), (136, 264)])
def test_linear_of_more_elements_than_32_bits_count(k, n):
    """The backward pass in one kernel and as separate ones: each row's dx, and dw of rows that are zeros but for the last ones."""
    from bioemu2_b200 import training as t

    rows = 2 ** 24 + 3001
    g = gen(43)
    w = (randn(g, n, k) / math.sqrt(k)).bfloat16()
    x = large(g, rows, k)
    y = t.linear_forward(x, w)[0]
    end = slice(rows - 700, rows)
    xd, wd = x[end].double(), w.double()
    want = xd @ wd.T
    check("y", y[end], want, 2 * U * (k + 2) * (xd.abs() @ wd.abs().T) + 1.01 * half(BF16) * want.abs() + tiny(BF16))
    del y
    dy = torch.zeros(rows, n, device=DEV, dtype=BF16)
    dy[end] = large(g, 700, n)
    dx, dw, db = t.linear_backward(dy, x, w)
    d = dy[end].double()
    want = d @ wd
    check("dx", dx[end], want, 2 * U * (n + 2) * (d.abs() @ wd.abs()) + 1.01 * half(BF16) * want.abs() + tiny(BF16))
    assert not dx[:end.start].any()
    # the zeros add nothing: 700 terms and their parts' sums
    want = d.T @ xd
    check("dw", dw, want, 2 * U * 1000 * (d.abs().T @ xd.abs()) + 1.01 * half(BF16) * want.abs() + tiny(BF16))
    check("db", db, d.sum(0), 1000 * U * d.abs().sum(0))


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,k,n", [(3000, 128, 512), (700, 200, 136)])
def test_linear_function_with_the_value_before_the_activation_in_fp32(act, rows, k, n):
    """The bias's gradient is then a sum in fp32 throughout: of dy times the slope at a, which is off by the product's rounding."""
    from bioemu2_b200 import training as t

    g, x, w = linear_inputs(rows, k, n, BF16)
    b, dy = randn(g, n), randn(g, rows, n).bfloat16()
    y, pre = t.linear_forward(x, w, b, act, save=F32)
    want = t.linear_backward(dy, x, w, pre, act)
    layer = t.Linear(k, n, activation=act, save_dtype=F32, device=DEV, dtype=BF16)
    with torch.no_grad():
        layer.weight.copy_(w)
        layer.bias.copy_(b)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    out = t.linear(*leaves, act, save_dtype=F32)
    out.backward(dy)
    assert torch.equal(out, y) and all(torch.equal(v.grad, u) for v, u in zip(leaves, want))
    a = x.double() @ w.double().T + b.double()
    off = 2 * U * (k + 2) * (x.double().abs() @ w.double().abs().T) + 2 * U * b.double().abs()
    slope = slope_oracle(a, act)
    if act == "relu":  # a step of one: within the product's rounding of zero a may have either sign and its slope be off by one, else by nothing
        off = (a.abs() <= off).double()
    terms = dy.double() * slope
    # the second derivatives are 1 at most; the slopes' own 16 U
    bound = (dy.double().abs() * (off + 16 * U) + (64 + rows / 64) * U * terms.abs()).sum(0)
    check("db", leaves[2].grad, terms.sum(0), bound + 2 * U * terms.sum(0).abs())
    xl = x.clone().requires_grad_()
    layer(xl).backward(dy)
    y2, pre2 = t.linear_forward(x, w, layer.bias.detach(), act, save=F32)
    assert all(torch.equal(u, v) for u, v in zip((xl.grad, layer.weight.grad), t.linear_backward(dy, x, w, pre2, act)))


def transition_step(t, leaves, z, dz):
    """Forward and backward of LN, a widening and a narrowing layer with the fp32 stream as residual; z's gradient and the parameters'."""
    z = z.detach().requires_grad_()
    x = t.layer_norm(z, leaves[0], leaves[1], out_dtype=BF16, checkpoint=True)
    h = t.linear(x, leaves[2], leaves[3], "silu", checkpoint=True)
    out = t.linear(h, leaves[4], None, None, z, checkpoint=True)
    return (out,) + torch.autograd.grad(out, (z, *leaves), dz)


def transition_leaves(g, d=128, hidden=512):
    w = [1 + 0.2 * randn(g, d), 0.2 * randn(g, d), (randn(g, hidden, d) / math.sqrt(d)).bfloat16(), 0.1 * randn(g, hidden),
         (randn(g, d, hidden) / math.sqrt(hidden)).bfloat16()]
    return [v.requires_grad_() for v in w]


def test_threads_with_streams_of_their_own():
    """Four threads train at the same time, a stream each: every result is the one that a thread alone gets."""
    import threading

    from bioemu2_b200 import training as t

    g = gen(51)
    leaves = transition_leaves(g)
    data = [(randn(g, 700 + 300 * i, 128), randn(g, 700 + 300 * i, 128)) for i in range(4)]
    want = [transition_step(t, leaves, *d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = transition_step(t, leaves, *data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors, errors
    assert all(torch.equal(a, b) for one, other in zip(got, want) for a, b in zip(one, other))


def test_under_autocast():
    """These calls take their types from their inputs: autocast changes nothing."""
    from bioemu2_b200 import training as t

    g = gen(52)
    leaves, z, dz = transition_leaves(g), randn(g, 900, 128), randn(g, 900, 128)
    want = transition_step(t, leaves, z, dz)
    for dtype in (BF16, F16):
        with torch.autocast("cuda", dtype=dtype):
            got = transition_step(t, leaves, z, dz)
        assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))


def test_captured_training_step():
    """Forward and backward of the differentiable functions in one graph, replayed with other inputs and other parameters."""
    from bioemu2_b200 import training as t

    g = gen(53)
    leaves, z, dz = transition_leaves(g), randn(g, 1300, 128), randn(g, 1300, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        transition_step(t, leaves, z, dz)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = transition_step(t, leaves, z, dz)
    for turn in range(3):
        with torch.no_grad():
            z.copy_(randn(g, 1300, 128))
            dz.copy_(randn(g, 1300, 128))
            leaves[2].mul_(1.01)
        graph.replay()
        want = transition_step(t, leaves, z, dz)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
