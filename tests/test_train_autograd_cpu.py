"""What autograd sees of the registered operators around a training step, on meta tensors: results through which no
gradient goes raise in a backward pass and on forward-mode tangents, and the Python functions return plain tensors."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from mhc_ops_b200 import mhc_orthogonalize, mhc_qk_norm_rope, mhc_qk_norm_rope_backward, mhc_qk_norm_rope_fn, ops

COEFFS = [1.5, -0.5, 0.0]


def _meta(*shape, grad=False):
    return torch.empty(*shape, device="meta", requires_grad=grad)


def _calls(q, g):
    k, f = _meta(1, 4, 2, 16), _meta(8)
    return {"qk_norm_rope": lambda: ops.qk_norm_rope(q, k, None, f, None, None, None, None, 1e-6, False),
            "qk_norm_rope_bwd": lambda: ops.qk_norm_rope_bwd(q, k, None, f, k, k, None, None, None, None, None, 1e-6,
                                                             False, True, True),
            "orthogonalize": lambda: ops.orthogonalize([g], COEFFS, 1e-7)}


@pytest.mark.parametrize("op", ["qk_norm_rope", "qk_norm_rope_bwd", "orthogonalize"])
def test_backward_through_a_registered_operator_raises(op):
    out = _calls(_meta(1, 4, 2, 16, grad=True), _meta(8, 64, grad=True))[op]()
    assert out[0].requires_grad
    with pytest.raises(RuntimeError, match="not implemented"):
        out[0].sum().backward()
    assert not _calls(_meta(1, 4, 2, 16), _meta(8, 64))[op]()[0].requires_grad


@pytest.mark.parametrize("op", ["qk_norm_rope", "qk_norm_rope_bwd", "orthogonalize"])
def test_forward_mode_tangents_raise(op):
    with fwd_ad.dual_level():
        dual = lambda *s: fwd_ad.make_dual(_meta(*s), _meta(*s))   # noqa: E731
        with pytest.raises((NotImplementedError, RuntimeError), match="forward AD"):
            _calls(dual(1, 4, 2, 16), dual(8, 64))[op]()


def test_python_functions_return_plain_tensors():
    q, k, f = _meta(1, 4, 2, 16, grad=True), _meta(1, 4, 2, 16), _meta(8)
    assert not any(t.requires_grad for t in mhc_qk_norm_rope(q, k, None, f))
    assert not mhc_qk_norm_rope_backward(q, k, None, f, k, k)[0].requires_grad
    assert not mhc_orthogonalize(_meta(8, 64, grad=True)).requires_grad
    assert mhc_qk_norm_rope_fn(q, k, None, f)[0].requires_grad


def test_autograd_function_traces_under_fake_tensors():
    """Both directions as single nodes, at a symbolic length."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def both(q, k, f, w, up):
        y = mhc_qk_norm_rope_fn(q, k, None, f, w)[0]
        return torch.autograd.grad(y, (q, w), up)

    args = (_meta(2, 5, 4, 16, grad=True), _meta(2, 5, 2, 16), _meta(8), _meta(16, grad=True), _meta(2, 5, 4, 16))
    graph = make_fx(both, tracing_mode="symbolic")(*args)
    names = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    assert sum("mhc.qk_norm_rope.default" in n for n in names) == 1
    assert sum("mhc.qk_norm_rope_bwd" in n for n in names) == 1


def test_coefficients_may_come_from_a_generator():
    from mhc_ops_b200.muon import _coeffs
    assert _coeffs((a, -0.5, 0.0) for a in (1.5, 2.0)) == [1.5, -0.5, 0.0, 2.0, -0.5, 0.0]
    with pytest.raises(ValueError, match="triples"):
        _coeffs(iter([(1.0, 2.0)]))
