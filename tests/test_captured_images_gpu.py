"""A captured transition replays on the weights it was captured with while the module goes on training (B200 only)."""

from __future__ import annotations

import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

from foldforge_b200 import _lib  # noqa: E402
from foldforge_b200.engine.capture import GraphedCall  # noqa: E402
from foldforge_b200.engine.modules import Transition  # noqa: E402

BF16 = torch.bfloat16


@pytest.mark.parametrize("frozen", [True, False])
@pytest.mark.parametrize("d,shape", [(128, (1, 20, 20)), (384, (1, 33)), (64, (3, 50))])
def test_replays_between_training_steps(d, shape, frozen):
    torch.manual_seed(d)
    module = Transition(d, 4).cuda()
    module.set_backend("b200")
    module.set_checkpoint("exact")
    for p in module.parameters():
        p.requires_grad_(not frozen)
    x = torch.randn(*shape, d, device="cuda").to(BF16)
    graphed = GraphedCall(module, [x])
    assert len(graphed.images) == 1
    want = graphed(x).clone()
    optimiser = None if frozen else torch.optim.SGD(module.parameters(), lr=0.1)
    for _ in range(3):
        xa = x.clone().requires_grad_()
        out = module(xa)
        out.float().square().mean().backward()
        if optimiser is not None:
            optimiser.step()
        with torch.no_grad():
            now = module(x)
        assert torch.equal(now, want) == frozen
        # memory that was let go is written over before the replay
        gc.collect()
        filled = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (1 << 18, 1 << 20, 1 << 22) for _ in range(8)]
        assert torch.equal(graphed(x), want)
        del filled
    again = GraphedCall(module, [x])
    assert torch.equal(again(x), now) and torch.equal(graphed(x), want)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def test_the_memory_of_a_replaced_image_waits_for_another_streams_reader():
    torch.manual_seed(0)
    module = Transition(128, 4).cuda()
    module.set_backend("b200")
    x = torch.randn(1, 20, 20, 128, device="cuda").to(BF16)
    with torch.no_grad():
        want = module(x)
        image = module._packed[1]
        address, size = image.data_ptr(), image.numel()
        del image
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)  # about 50 ms
            got = module(x)
        module.squeeze.weight.mul_(2.0)
        module(x)  # replaces the image
        others = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(8)]
        assert not side.query() and address not in [t.data_ptr() for t in others]
        side.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
