"""What may not happen while a training step is captured into a graph."""
import gc
import weakref

import pytest
import torch

import music_generator_amd as M
from music_generator_amd import task


@pytest.mark.gpu
def test_nothing_is_collected_while_a_step_is_captured():
    """A dropped model that a reference cycle keeps alive (a callback's closure is enough) holds captured graphs and pinned
    buffers: they are destroyed before the capture of another model's step begins, never inside it."""
    real = torch.rand((4, 4, 750, 2), generator=torch.Generator().manual_seed(1)).cuda() * 2 - 1

    def trained(steps):
        M.clear_session()
        gan = task.build(1)[2][0][0]
        gan.seed(3)
        gan.use_graph = True
        for _ in range(steps):
            gan.train_step(real)
        torch.cuda.synchronize()
        return gan

    class Holder:
        pass

    old = Holder()
    old.gan, old.itself = trained(3), old
    entry = next(iter(old.gan._graphs.values()))
    gone = weakref.ref(entry["graph"])
    del entry
    gc.disable()                      # the collector runs when the capture asks for it
    try:
        del old
        gc.enable()
        gan, seen = trained(1), []
        body = gan._step_body
        gan._step_body = lambda batch: (seen.append((torch.cuda.is_current_stream_capturing(), gc.isenabled(), gone() is None)), body(batch))[1]
        for _ in range(3):
            gan.train_step(real)
        torch.cuda.synchronize()
        assert seen == [(True, False, True)] and gc.isenabled()
        gc.disable()
        again = trained(1)            # a program that has switched the collector off keeps it off
        again.train_step(real)
        torch.cuda.synchronize()
        assert not gc.isenabled()
    finally:
        gc.enable()
