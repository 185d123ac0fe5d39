"""The stream that a workspace of Runner.call_prefix_paged is allocated for is the one that the call runs on, so that
torch's allocator hands it on in that stream's order."""
from types import SimpleNamespace

import pytest

from tests.conftest import load_package


def test_allocation_stream_of_a_handle():
    cuda = SimpleNamespace(default_stream=lambda: "default", ExternalStream=lambda handle: ("external", handle))
    of = lambda stream: load_package().Runner._allocation_stream(SimpleNamespace(cuda=cuda), stream)
    assert of(None) is None and of(0) == "default" and of(0x1234) == ("external", 0x1234)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["current", "side", "default", "default_beside_a_side_stream"])
def test_workspace_belongs_to_the_stream_of_its_call(gpu_runner, which):
    import torch
    from tests.serving import Batch
    x = Batch(8, 2, 64, [(256, [(1, 300), (1, 257)])])
    o, l = x.outputs(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    handle = {"current": None, "side": side.cuda_stream}.get(which, torch.cuda.default_stream().cuda_stream)
    with torch.cuda.stream(side if which == "default_beside_a_side_stream" else None):
        ws = x.attend(gpu_runner, o, l, 0, stream=handle)
    torch.cuda.synchronize()
    x.check(o, l, 0)
    at = ws.data_ptr()
    segment, = [s for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"]]
    assert segment["stream"] == (0 if handle is None else handle)
