"""What the training operators refuse, before anything is launched or allocated on a device (no GPU needed)."""
import pytest
import torch

from bioemu2_b200 import _lib, training as t

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def z(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def kept(*shape, dtype=F32, values=torch.float8_e4m3fn, exponents=torch.uint8, groups=None):
    groups = (shape[-1] + 31) // 32 if groups is None else groups
    return t.Checkpoint8(z(*shape).to(values), z(*shape[:-1], groups).to(exponents), dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: t.checkpoint8(z(3, 4, dtype=torch.float64)), "x must be float32"),
    (lambda: t.checkpoint8(z(3, 4).int()), "x must be float32"),
    (lambda: t.checkpoint8(torch.tensor(1.0)), "at least one column"),
    (lambda: t.checkpoint8(z(3, 0)), "at least one column"),
    (lambda: kept(3, 64).restore(torch.float64), "restored activation"),
    (lambda: kept(3, 64, values=torch.uint8).restore(), "float8_e4m3fn with uint8"),
    (lambda: kept(3, 64, exponents=torch.int32).restore(), "float8_e4m3fn with uint8"),
    (lambda: kept(3, 65, groups=2).restore(), "exponents have shape"),
    (lambda: kept(3, 64, groups=3).restore(), "exponents have shape"),
    (lambda: kept(3, 0, groups=0).restore(), "at least one column"),
], ids=range(10))
def test_checkpoints(call, match):
    with pytest.raises(ValueError, match=match):
        call()


NORM = dict(dy=z(5, 8), x=z(5, 8), mean=z(5), rstd=z(5), weight=z(8))


@pytest.mark.parametrize("call,match", [
    (lambda: t.layer_norm_forward(z(2, 8193)), "1 to 8192 columns"),
    (lambda: t.layer_norm_forward(z(2, 0)), "1 to 8192 columns"),
    (lambda: t.layer_norm_forward(torch.tensor(1.0)), "1 to 8192 columns"),
    (lambda: t.layer_norm_forward(z(2, 8, dtype=torch.float64)), "x must be"),
    (lambda: t.layer_norm_forward(z(2, 8), out_dtype=torch.float64), "y must be"),
    (lambda: t.layer_norm_forward(z(2, 8, dtype=BF16), out_dtype=F32), "wants x in float32"),
    (lambda: t.layer_norm_forward(z(2, 8, dtype=BF16), out_dtype=F16), "wants x in float32"),
    (lambda: t.layer_norm_forward(z(2, 8), z(7)), "weight has shape"),
    (lambda: t.layer_norm_forward(z(2, 8), z(8, 1)), "weight has shape"),
    (lambda: t.layer_norm_forward(z(2, 8), None, z(9)), "bias has shape"),
    (lambda: t.layer_norm_forward(z(2, 8), z(8).int()), "weight must be"),
    (lambda: t.layer_norm_backward(**{**NORM, "dy": z(5, 9)}), "dy has shape"),
    (lambda: t.layer_norm_backward(**{**NORM, "dy": z(4, 8)}), "dy has shape"),
    (lambda: t.layer_norm_backward(**{**NORM, "x": z(5, 8, dtype=BF16)}), "wants x in float32"),
    (lambda: t.layer_norm_backward(**{**NORM, "x": kept(5, 8, dtype=BF16)}), "wants x in float32"),
    (lambda: t.layer_norm_backward(**{**NORM, "x": kept(5, 8, groups=2)}), "exponents have shape"),
    (lambda: t.layer_norm_backward(**{**NORM, "mean": z(4)}), "mean and rstd"),
    (lambda: t.layer_norm_backward(**{**NORM, "mean": z(5, 1)}), "mean and rstd"),
    (lambda: t.layer_norm_backward(**{**NORM, "rstd": z(5, dtype=BF16)}), "mean and rstd"),
    (lambda: t.layer_norm_backward(**{**NORM, "weight": z(9)}), "weight has shape"),
    (lambda: t.layer_norm_backward(**NORM, grad_dtype=torch.float64), "parameters' gradient"),
    (lambda: t.LayerNorm((4, 8)), "last axis alone"),
    (lambda: t.LayerNorm(9000), "last axis alone"),
    (lambda: t.LayerNorm(8)(z(2, 9)), "its last axis must be 8"),
], ids=range(24))
def test_layer_norm(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def b(*shape):
    return z(*shape, dtype=BF16)


@pytest.mark.parametrize("call,match", [
    (lambda: t.linear_forward(z(2, 8), z(16, 8)), "both be bfloat16 or both float16"),
    (lambda: t.linear_forward(b(2, 8), z(16, 8, dtype=F16)), "both be bfloat16 or both float16"),
    (lambda: t.linear_forward(b(2, 8), b(16, 16)), "does not match"),
    (lambda: t.linear_forward(b(2, 8), b(8)), "does not match"),
    (lambda: t.linear_forward(torch.tensor(1.0, dtype=BF16), b(8, 8)), "does not match"),
    (lambda: t.linear_forward(b(2, 12), b(16, 12)), "multiples of 8"),
    (lambda: t.linear_forward(b(2, 8), b(12, 8)), "multiples of 8"),
    (lambda: t.linear_forward(b(2, 8), b(0, 8)), "multiples of 8"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), activation="tanh"), "activation must be one of"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), out_dtype=F16), "y is"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), residual=b(2, 8)), "residual is"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), residual=b(1, 16)), "residual is"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), residual=z(2, 16), out_dtype=BF16), "residual is"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), residual=z(2, 16, dtype=F16)), "y is"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), save=F16), "saved as"),
    (lambda: t.linear_forward(b(2, 8), b(16, 8), z(8)), "bias has shape"),
    (lambda: t.linear_backward(b(2, 16), None, b(16, 8)), "wants x"),
    (lambda: t.linear_backward(b(2, 8), b(2, 8), b(16, 8)), "dy must be"),
    (lambda: t.linear_backward(z(2, 16, dtype=F16), b(2, 8), b(16, 8)), "dy must be"),
    (lambda: t.linear_backward(b(3, 16), b(2, 8), b(16, 8)), "dy must be"),
    (lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8), None, "silu"), "pre must be"),
    (lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8), b(2, 8), "silu"), "pre must be"),
    (lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8), z(2, 16, dtype=F16), "silu"), "pre must be"),
    (lambda: t.linear_backward(b(2, 16), kept(2, 8, dtype=F32), b(16, 8)), "both be bfloat16"),
    (lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8), activation="Silu"), "activation must be one of"),
    (lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8), bias_dtype=torch.float64), "bias's gradient"),
    (lambda: t.Linear(12, 8), "multiples of 8"),
    (lambda: t.Linear(8, 8, activation="swish"), "activation must be one of"),
], ids=range(28))
def test_linear(call, match):
    with pytest.raises(ValueError, match=match):
        call()


@pytest.mark.parametrize("call", [
    lambda: t.checkpoint8(z(3, 4)),
    lambda: kept(3, 64).restore(),
    lambda: t.layer_norm(z(3, 8), z(8), z(8)),
    lambda: t.layer_norm_backward(**NORM),
    lambda: t.linear(b(2, 8), b(16, 8), z(16), "gelu", b(2, 16)),
    lambda: t.linear_backward(b(2, 16), b(2, 8), b(16, 8)),
    lambda: t.LayerNorm(8)(z(2, 8)),
    lambda: t.Linear(8, 16)(b(2, 8)),
], ids=range(8))
def test_host_tensors(call):
    """Everything about the call is right but where its tensors are: there is no CPU path."""
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call()


def test_modules_hold_the_parameters_of_their_namesakes():
    assert set(t.LayerNorm(8).state_dict()) == set(torch.nn.LayerNorm(8).state_dict())
    assert set(t.Linear(8, 16).state_dict()) == set(torch.nn.Linear(8, 16).state_dict())
    t.Linear(8, 16).load_state_dict(torch.nn.Linear(8, 16).state_dict())
    assert t.Linear(8, 16, bias=False).bias is None and t.LayerNorm(8, bias=False).bias is None


def test_status_codes_become_exceptions():
    """The extension raises through the binding's own check: a failed library call is the exception it always was."""
    with pytest.raises(ValueError):
        _lib.check(_lib.ERR_INVALID_ARGUMENT)
    with pytest.raises(_lib.DeviceWaitError):
        _lib.check(_lib.ERR_DEVICE_WAIT)


def test_dtensors_are_refused():
    """A DTensor has no memory of its own: its null pointer would stand for a parameter that was not given."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, distribute_tensor

    mine = not dist.is_initialized()
    if mine:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        d = lambda v: distribute_tensor(v, mesh, [Replicate()])  # noqa: E731
        for call in (lambda: t.layer_norm(z(2, 8), d(z(8)), z(8)), lambda: t.layer_norm(z(2, 8), z(8), d(z(8))), lambda: t.layer_norm(d(z(2, 8)), z(8)),
                     lambda: t.layer_norm(z(2, 8), d(z(8)).requires_grad_()), lambda: t.layer_norm_backward(**{**NORM, "weight": d(z(8))}),
                     lambda: t.linear(b(2, 8), b(16, 8), d(z(16))), lambda: t.linear(b(2, 8), b(16, 8), None, None, d(b(2, 16))),
                     lambda: t.linear(b(2, 8), d(b(16, 8))), lambda: t.linear(d(b(2, 8)), b(16, 8)), lambda: t.checkpoint8(d(z(2, 8)))):
            with pytest.raises(ValueError, match="memory of its own"):
                call()
    finally:
        if mine:
            dist.destroy_process_group()


@pytest.mark.parametrize("call", [
    lambda d: t.layer_norm(d(z(2, 8)), z(8), z(8)),
    lambda d: t.layer_norm(z(2, 8), d(z(8)), z(8)),
    lambda d: t.layer_norm(z(2, 8), z(8), d(z(8))),
    lambda d: t.layer_norm(z(2, 8).requires_grad_(), d(z(8))),
    lambda d: t.LayerNorm(8)(d(z(2, 8))),
    lambda d: t.linear(d(b(2, 8)), b(16, 8)),
    lambda d: t.linear(b(2, 8), d(b(16, 8))),
    lambda d: t.linear(b(2, 8), b(16, 8), d(z(16))),
    lambda d: t.linear(b(2, 8), b(16, 8), None, "silu", d(b(2, 16))),
    lambda d: t.Linear(8, 16)(d(b(2, 8))),
], ids=range(10))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(call, grad):
    """A result without a tangent would read as a derivative of zero, with and without gradients in the other mode."""
    from torch.autograd import forward_ad

    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(lambda v: forward_ad.make_dual(v, torch.ones_like(v)))


def wide(cols, dtype, rows=None):
    return torch.empty(1, dtype=dtype).expand(*([] if rows is None else [rows]), cols)


@pytest.mark.parametrize("call,match", [
    (lambda: t.checkpoint8(wide(2 ** 31, BF16)), "at most 2147483647"),
    (lambda: t.checkpoint8(wide(2 ** 32 + 8, F32, 3)), "at most 2147483647"),
    (lambda: t.Checkpoint8(wide(2 ** 32 + 8, torch.float8_e4m3fn), wide(2 ** 27 + 1, torch.uint8), F32).restore(), "at most 2147483647"),
    (lambda: t.linear_forward(wide(2 ** 32 + 8, BF16, 2), wide(2 ** 32 + 8, BF16, 16)), "at most 16777216"),
    (lambda: t.linear_forward(b(2, 8), wide(8, BF16, 2 ** 32 + 8)), "at most 16777216"),
    (lambda: t.linear_backward(wide(2 ** 32 + 8, BF16, 2), b(2, 8), wide(8, BF16, 2 ** 32 + 8)), "at most 16777216"),
], ids=range(6))
def test_widths_that_the_library_does_not_count(call, match):
    """Taken modulo 2^32 they would be narrow rows: a prefix would be computed and the rest left as it was allocated."""
    with pytest.raises(ValueError, match=match):
        call()


def test_widest_rows_of_a_checkpoint():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        t.checkpoint8(wide(2 ** 31 - 1, BF16))


def test_type_of_the_value_before_the_activation():
    for dtype in (F16, torch.float64):
        with pytest.raises(ValueError, match="saved as"):
            t.linear(b(2, 8), b(16, 8), activation="silu", save_dtype=dtype)
        with pytest.raises(ValueError, match="saved as"):
            t.Linear(8, 16, activation="silu", save_dtype=dtype)(b(2, 8))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        t.linear(b(2, 8), b(16, 8).requires_grad_(), activation="silu", save_dtype=F32)


def test_modules_pickled_without_the_type_of_the_value_before_the_activation():
    layer = t.Linear(8, 16, dtype=BF16)
    del layer.__dict__["save_dtype"]
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer(b(2, 8))


def test_inference_mode_goes_the_same_way():
    with torch.inference_mode(), pytest.raises(RuntimeError, match="CUDA tensors only"):
        t.layer_norm(z(2, 8), z(8), z(8))
