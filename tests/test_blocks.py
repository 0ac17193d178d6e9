"""CPU tests of the conditioned image block's host side (blocks.py)."""
import pytest
import torch

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
