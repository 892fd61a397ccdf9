"""The status calls of the quantised libraries answer for everything launched so far, on side streams too."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", ["kernels", "prefill_mq"])
def test_device_status_waits_for_side_streams(module):
    import importlib
    m = importlib.import_module("flagrot_releaser_b200." + module)
    m.device_status()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            torch.cuda._sleep(400_000_000)                     # a fifth of a second
    assert not any(s.query() for s in streams), "the streams ended too soon for this test"
    assert m.device_status() == 0
    assert all(s.query() for s in streams)
