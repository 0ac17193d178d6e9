"""CPU tests of the conditioned image block's host side (blocks.py)."""
import pytest
import torch
from torch.autograd import forward_ad

WHOLE = [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32, torch.uint64]


@pytest.mark.parametrize("dtype", WHOLE)
@pytest.mark.parametrize("states", [5, 300, 70000, 2 ** 31 - 1])
def test_lengths_of_every_whole_type(dtype, states):
    """Every type of whole numbers is taken whatever the number of states, and no
    value wraps on its way to 32 bits."""
    from rdv_project_b200.blocks import _key_lengths

    info = torch.iinfo(dtype)
    values = [0, 1, 100, info.max, max(info.min, -2 ** 63), max(info.min, -7), min(info.max, 2 ** 32 + 3)]
    got = _key_lengths(torch.tensor(values, dtype=dtype), len(values), states)
    assert got.dtype == torch.int32 and got.is_contiguous()
    # below 0 and above the states: as 0 and as the states, by the kernels if not here
    assert [min(max(n, 0), states) for n in got.tolist()] == [min(max(n, 0), states) for n in values]


def test_lengths_refusals():
    from rdv_project_b200.blocks import _key_lengths

    for bad in (torch.zeros(2), torch.zeros(2, dtype=torch.bool), torch.zeros(2, dtype=torch.complex64),
                torch.zeros(3, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int64), torch.tensor(3)):
        with pytest.raises(ValueError):
            _key_lengths(bad, 2, 9)


def test_forward_mode_inputs_are_refused():
    """A tangent is not dropped in silence, with gradients enabled or not."""
    import rdv_project_b200 as rdv

    x, w, q = torch.ones(2, 3, 8), torch.ones(8), torch.ones(1, 2, 2, 8)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: rdv.group_norm(dual(x), 2), lambda: rdv.group_norm(x, 2, dual(w)),
                     lambda: rdv.group_norm(x, 2, w, dual(w)), lambda: rdv.cross_attention(dual(q), q, q),
                     lambda: rdv.cross_attention(q, dual(q), q), lambda: rdv.cross_attention(q, q, dual(q)),
                     lambda: rdv.dropout(dual(x), 0.1, 0), lambda: rdv.dropout(x, 0.1, 0, residual=dual(x))):
            for enabled in (True, False):
                with torch.set_grad_enabled(enabled), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


def test_wrapped_inputs_ask_for_gradients_like_their_tensors():
    import rdv_project_b200 as rdv
    from rdv_project_b200.blocks import _wants_grad

    x = torch.ones(2, 8)
    wrapped = rdv.wrap(x.clone().requires_grad_())
    assert _wants_grad(None, wrapped) and not _wants_grad(rdv.wrap(x), None)
    with torch.no_grad():
        assert not _wants_grad(wrapped)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        _wants_grad(rdv.wrap(forward_ad.make_dual(x, x)))
