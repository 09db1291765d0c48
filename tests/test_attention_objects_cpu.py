"""PagedKV and SequenceBatch keep addresses of their tensors: what they hold is not exchanged afterwards."""
import pytest


@pytest.fixture(scope="module")
def op(sgq):
    import soverign_grad_amd.attention as attention

    return attention


@pytest.mark.parametrize("name", ["PagedKV", "SequenceBatch"])
def test_attributes_are_not_assigned(op, name):
    cls = getattr(op, name)
    x = cls.__new__(cls)
    for attr in cls.__slots__:
        with pytest.raises(AttributeError, match="make a new one"):
            setattr(x, attr, 1)
        with pytest.raises(AttributeError, match="make a new one"):
            delattr(x, attr)
