"""``_native.current_stream_ptr`` takes a device in each of torch's ways."""
import pytest
import torch


@pytest.mark.gpu
def test_current_stream_of_a_device_in_any_form():
    from efficient_probing_amd import _native as N
    want = torch.cuda.current_stream("cuda:0").cuda_stream
    side = torch.cuda.Stream()
    for d in (None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda:0"), torch.device("cuda", 0)):
        assert N.current_stream_ptr(d) == want
        with torch.cuda.stream(side):
            assert N.current_stream_ptr(d) == side.cuda_stream


def test_device_index_of_any_form():
    from efficient_probing_amd import _native as N
    assert [N._device_index(d) for d in (None, 2, "cuda", "cuda:3", torch.device("cuda"), torch.device("cuda", 1))] == [None, 2, None, 3, None, 1]
