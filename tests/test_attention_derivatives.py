"""Which derivatives the packed attention entry points give, and which they refuse: none is dropped without an error."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from astrai_b200.ops import flash, native


@pytest.fixture
def raw_kernel(monkeypatch):
    """The operator as it is on a GPU: it works on the data, so nothing that is differentiated passes through it."""
    monkeypatch.setattr(native, "require", lambda: torch.ops.astrai_b200)

    def flash_fwd(q, k, v, cu_q, cu_k, batch, sq, sk, max_q, causal, scale):
        return torch.from_numpy(fwAD.unpack_dual(q).primal.detach().float().numpy().copy()), torch.zeros(q.shape[0], q.shape[1])

    monkeypatch.setattr(torch.ops.astrai_b200, "flash_fwd", flash_fwd, raising=False)


def _rows(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape)))


CU = torch.tensor([0, 2, 5], dtype=torch.int32)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_through_the_ragged_entry_is_refused(raw_kernel, which):
    rows = [_rows(5, 2, 64) for _ in range(3)]
    with fwAD.dual_level():
        rows[which] = fwAD.make_dual(rows[which], _rows(5, 2, 64))
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
            flash.flash_attention_varlen(*rows, CU, CU, 3, 3)
    assert flash.flash_attention_varlen(*[fwAD.unpack_dual(r).primal for r in rows], CU, CU, 3, 3).shape == (5, 2, 64)


def test_reverse_mode_through_the_ragged_entry_is_recorded(raw_kernel):
    q, k, v = (_rows(5, 2, 64) for _ in range(3))
    assert flash.flash_attention_varlen(q.requires_grad_(), k, v, CU, CU, 3, 3).requires_grad
    with torch.no_grad():
        assert not flash.flash_attention_varlen(q, k, v, CU, CU, 3, 3).requires_grad


def test_a_serving_step_goes_straight_to_the_kernel_and_drops_no_derivative(raw_kernel):
    q, k, v = (_rows(5, 2, 64) for _ in range(3))
    assert flash.flash_attention_ragged(q, k, v, CU, CU, 3, 3, 0.125).grad_fn is None
    with fwAD.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
            flash.flash_attention_ragged(fwAD.make_dual(q, _rows(5, 2, 64)), k, v, CU, CU, 3, 3, 0.125)
        assert flash.flash_attention_ragged(q, k, v, CU, CU, 3, 3, 0.125).shape == (5, 2, 64)
    q.requires_grad_()
    assert flash.flash_attention_ragged(q, k, v, CU, CU, 3, 3, 0.125).requires_grad
    with torch.inference_mode():
        assert flash.flash_attention_ragged(q, k, v, CU, CU, 3, 3, 0.125).grad_fn is None
