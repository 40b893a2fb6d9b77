"""A packed weight image that a captured graph reads (by its address alone) outlives training passes and
changed weights; the prepare calls and the kernels have stand-ins here, so that no GPU is needed."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch
from torch import nn

from foldforge_b200 import kernels
from foldforge_b200.engine import capture, dit, modules
from foldforge_b200.engine.modules import Transition


@pytest.fixture
def packs(monkeypatch):
    """CPU tensors pass for ones on an sm_100 device; an image is a copy of the squeeze weight, and the kernel
    returns its input plus the image's sum. The list gets a weak reference to every image made."""
    made = []

    def prepare(weights, *_):
        image = weights["squeeze.weight"].clone()
        made.append(weakref.ref(image))
        return image

    def run(x, *args, **_):
        return x + next(a for a in args if a is not None and a.dim() == 2 and a.dtype == torch.float32).sum().to(x.dtype)

    monkeypatch.setattr(modules, "_device_reason", lambda *ts: None)
    monkeypatch.setattr(modules, "_library_reason", lambda: None)
    for name in ("transition_prepare", "single_transition_prepare", "transition_gemm_prepare"):
        monkeypatch.setattr(kernels, name, prepare)
    for name in ("transition", "single_transition", "transition_gemm"):
        monkeypatch.setattr(kernels, name, run)
    return made


def alive(made) -> list[bool]:
    gc.collect()
    return [ref() is not None for ref in made]


def captured(monkeypatch, module, x):
    """A call that believes a graph is being captured."""
    with monkeypatch.context() as m, torch.no_grad():
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        return module(x)


def op(d, n=4):
    module = Transition(d, n)
    module.set_backend("b200")
    module.set_checkpoint("exact")
    return module


CASES = [(128, (1, 3, 3)), (384, (1, 3)), (64, (2, 5))]


@pytest.mark.parametrize("frozen", [True, False])
@pytest.mark.parametrize("d,shape", CASES)
def test_a_captured_image_outlives_training_passes(packs, monkeypatch, d, shape, frozen):
    module = op(d)
    for p in module.parameters():
        p.requires_grad_(not frozen)
    x = torch.randn(*shape, d).to(torch.bfloat16)
    with torch.no_grad():
        module(x)  # the eager call before a capture
    captured(monkeypatch, module, x)
    assert alive(packs) == [True]
    for _ in range(2):
        module(x.clone().requires_grad_())
        assert alive(packs)[0]
    with torch.no_grad():
        module.squeeze.weight.mul_(2.0)  # a step of an optimiser
    module(x.clone().requires_grad_())
    with torch.no_grad():
        module(x)
        module(x)
    assert alive(packs)[0]


@pytest.mark.parametrize("d,shape", CASES)
def test_training_passes_leave_the_image_of_frozen_weights_alone(packs, d, shape):
    """Another stream or thread may be reading it: a gradient of the input alone replaces nothing."""
    module = op(d)
    for p in module.parameters():
        p.requires_grad_(False)
    x = torch.randn(*shape, d).to(torch.bfloat16)
    with torch.no_grad():
        module(x)
    module(x.clone().requires_grad_())
    with torch.no_grad():
        module(x)
    assert alive(packs)[0] and module._packed[1] is packs[0]()


@pytest.mark.parametrize("d,shape", CASES)
def test_passes_see_weights_changed_through_data(packs, d, shape):
    """``p.data`` leaves a parameter's version as it was: the passes that train and the first one without
    gradients after them see the new weights all the same, frozen ones too where a gradient is formed."""
    module = op(d)
    x = torch.randn(*shape, d).to(torch.bfloat16)

    def want():
        return x + module.squeeze.weight.detach().sum().to(x.dtype)

    with torch.no_grad():
        assert torch.equal(module(x), want())
    for _ in range(2):
        module.squeeze.weight.data.mul_(-3.0)
        assert torch.equal(module(x.clone().requires_grad_()), want())
    module.squeeze.weight.data.mul_(-3.0)
    with torch.no_grad():
        assert torch.equal(module(x), want())
    for p in module.parameters():
        p.requires_grad_(False)
    module.squeeze.weight.data.mul_(-3.0)
    assert torch.equal(module(x.clone().requires_grad_()), want())


def test_the_cache_may_change_between_the_look_and_the_return(packs):
    """As another thread's call may do it."""
    module = op(128)
    x = torch.randn(1, 3, 3, 128).to(torch.bfloat16)

    class Key:
        def __ne__(self, key):  # the look
            module._packed = None
            return False

    with torch.no_grad():
        module(x)
        module._packed = (Key(), module._packed[1])
        assert torch.equal(module(x), x + module.squeeze.weight.sum().to(x.dtype))


def test_an_image_packed_under_capture_stays_with_the_graph(packs, monkeypatch):
    """Its contents are there once the graph has run, so the calls outside it make their own."""
    module = op(128)
    x = torch.randn(1, 3, 3, 128).to(torch.bfloat16)
    captured(monkeypatch, module, x)
    assert module._packed is None
    with torch.no_grad():
        module(x)
    assert alive(packs) == [True, True] and module._packed[1] is packs[1]()


def test_a_holder_takes_the_images_in_place_of_the_module(packs, monkeypatch):
    """What a capture holds goes with it; without a holder the images stay as long as the module."""
    module, kept = op(128), []
    x = torch.randn(1, 3, 3, 128).to(torch.bfloat16)
    with torch.no_grad():
        module(x)
    with capture.holding(kept):
        captured(monkeypatch, module, x)
        captured(monkeypatch, module, x)
    assert len(kept) == 1 and kept[0] is packs[0]()
    with torch.no_grad():
        module.squeeze.weight.mul_(2.0)
        module(x)
    assert alive(packs) == [True, True]
    kept.clear()
    assert alive(packs) == [False, True]
    captured(monkeypatch, module, x)
    with torch.no_grad():
        module.squeeze.weight.mul_(2.0)
        module(x)
    assert alive(packs) == [False, True, True]
    del module
    assert alive(packs) == [False, False, False]


def test_a_captured_image_of_the_token_transformer_outlives_changed_weights(monkeypatch):
    made = []

    def prepare(weights, *_):
        made.append(weakref.ref(image := torch.zeros(4)))
        return image

    monkeypatch.setattr(kernels, "dit_prepare", prepare)
    block = dit.TokenDiT.__new__(dit.TokenDiT)
    nn.Module.__init__(block)
    block.weight, block._packed = nn.Parameter(torch.zeros(2)), None
    block._pack(torch.device("cpu"))
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        block._pack(torch.device("cpu"))
    with torch.no_grad():
        block.weight.add_(1.0)
    block._pack(torch.device("cpu"))
    assert alive(made) == [True, True]


def test_an_image_is_recorded_on_the_streams_that_read_it(packs, monkeypatch):
    """So that the memory of one that is replaced waits for them; a captured one is held instead."""

    class Image:
        def __init__(self):
            self.streams = []

        def get_device(self):
            return 0

        def record_stream(self, stream):
            self.streams.append(stream)

    module, image = op(128), Image()
    for stream in ("one", "two", "one"):
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device, s=stream: s)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index, s=stream: hash(s), raising=False)
        assert module._cached_pack(lambda weights: image) is image
    assert image.streams == ["one", "two"]
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        module._cached_pack(lambda weights: image)
    assert len(image.streams) == 2
