"""What the device-pointer calls take for an address, without a GPU: nothing that lies in host memory gets as far as a kernel."""
import numpy as np
import pytest
import torch

import exactinfer_b200 as e


@pytest.mark.parametrize("bad", (torch.zeros(4), torch.zeros(1, dtype=torch.int32)))
def test_host_tensors_are_refused(bad):
    with pytest.raises(ValueError):
        e._ptr(bad)
    with pytest.raises(ValueError):
        e.KvBatch(1, 1, 1, 1, 4096, 4096, bad, 1)
    with pytest.raises(ValueError):
        e.beam_select(bad, 4, 1, 1, 4096, 1, 4096, 4096, 4096, 4096, 1 << 20)


@pytest.mark.parametrize("bad", (np.array([4096]), np.array([4096.0]), np.zeros(4, np.int32), 4096.0, "4096", [4096]))
def test_no_number_is_made_of_arrays_and_the_like(bad):
    """An array of one element would have passed as the address that its element says."""
    with pytest.raises(TypeError):
        e._ptr(bad)


def test_addresses_are_taken_as_they_are():
    class Tensor:
        def data_ptr(self):
            return 4096

    assert e._ptr(None) is None and e._ptr(4096) == 4096 and e._ptr(np.int64(4096)) == 4096 and e._ptr(Tensor()) == 4096
