"""CPU: what the Python functions of the attention-side layers refuse or resolve before they call the library.  CPU tensors pass as those
of the current GPU, and the library is one that no call may reach."""
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


class Unreachable:
    def __getattr__(self, name):
        raise AssertionError("%s was called" % name)


@pytest.fixture
def L(monkeypatch):
    from yolo_amd import _lib
    from yolo_amd.utils import layer_utils
    monkeypatch.setattr(layer_utils, "_gpu", lambda: -1)                            # get_device() of a CPU tensor
    monkeypatch.setattr(_lib, "lib", Unreachable)
    layer_utils._attention_workspace.cache_clear()
    yield layer_utils
    layer_utils._attention_workspace.cache_clear()


def refused(call, text):
    with pytest.raises(ValueError, match=text):
        call()


def huge(*shape):
    """A tensor of more than 2^31 along one dimension; its pages are never touched."""
    return torch.empty(shape, dtype=BF16)


def test_sizes_past_32_bits_are_refused(L):
    """The C entries take int sizes, and ctypes passes the low 32 bits of a longer one: 2^32 + 8 would run as 8."""
    n = 2 ** 32 + 8
    refused(lambda: L.linear(huge(1, n), huge(1, n)), "2\\^31")
    refused(lambda: L.linear(huge(2, 1), huge(n, 1)), "2\\^31")
    one = huge(1, 1, 1, 8)
    refused(lambda: L.cross_attention(one, huge(1, n, 1, 1).expand(1, n, 1, 8), huge(1, n, 1, 1).expand(1, n, 1, 8)), "2\\^31")
    refused(lambda: L.cross_attention(huge(1, n, 1, 1), huge(1, 1, 1, 1), huge(1, 1, 1, 1)), "2\\^31")
    refused(lambda: L.cross_attention(huge(1, 1, n, 1), huge(1, 1, 1, 1), huge(1, 1, 1, 1)), "2\\^31")
    refused(lambda: L.cross_attention(huge(n, 1, 1, 1), huge(n, 1, 1, 1), huge(n, 1, 1, 1)), "2\\^31")
    refused(lambda: L.cross_attention(huge(1, 1, 1, n), huge(1, 1, 1, n), huge(1, 1, 1, n)), "2\\^31")
    refused(lambda: L.qk_norm_rope(huge(n, 1, 1, 1), None), "2\\^31")
    refused(lambda: L.qk_norm_rope(huge(1, n, 1, 1), None), "2\\^31")
    refused(lambda: L.qk_norm_rope(huge(1, 1, n, 1), None), "2\\^31")
    refused(lambda: L.qk_norm_rope(huge(1, 1, 1, n), None), "2\\^31")
    refused(lambda: L.qk_norm_rope(one, huge(1, n, 1, 1).expand(1, n, 1, 8)), "2\\^31")
    refused(lambda: L.qk_norm_rope(one, huge(1, 1, n, 1).expand(1, 1, n, 8)), "2\\^31")


def test_lazily_negated_tensors_hold_their_values(L):
    """The imaginary part of a conjugate is a view with torch's negative bit: its memory holds the values' negatives."""
    z = torch.complex(torch.arange(8.0), torch.arange(8.0) + 1)
    x = torch.conj(z).imag
    assert x.is_neg()
    got = L._dev(x, "x", -1)
    assert not got.is_neg() and torch.equal(got, -(torch.arange(8.0) + 1))
    same = torch.arange(8.0)
    assert L._dev(same, "x", -1) is same


def test_forward_mode_derivatives_are_refused(L):
    """A dual tensor of torch.autograd.forward_ad would come out without its tangent.  Like requires_grad it is refused, for every operand;
    plain tensors inside a dual level are not."""
    from torch.autograd import forward_ad
    x, w, b = torch.randn(3, 8), torch.randn(4, 8), torch.randn(4)
    q, k = torch.randn(1, 2, 2, 8), torch.randn(1, 3, 1, 8)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for i in range(4):
            a = [x, w, b, torch.randn(3, 4)]
            a[i] = dual(a[i])
            refused(lambda: L.linear(a[0], a[1], a[2], residual=a[3]), "tangent")
            with torch.no_grad():
                refused(lambda: L.linear(a[0], a[1], a[2], residual=a[3]), "tangent")
        for i in range(3):
            a = [q, k, k.clone()]
            a[i] = dual(a[i])
            refused(lambda: L.cross_attention(*a), "tangent")
        n = torch.ones(8)
        for i in range(4):
            a = [q, k, n, n.clone()]
            a[i] = dual(a[i])
            refused(lambda: L.qk_norm_rope(*a), "tangent")
        with pytest.raises(AssertionError, match="yolo_linear was called"):
            L.linear(x, w, b)
