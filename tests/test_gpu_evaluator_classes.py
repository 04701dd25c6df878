"""Fitting on class numbers: heads and labels that the cross entropy without logits meets through the evaluator."""
import numpy as np
import pytest
import torch

import music_generator_amd as M
from music_generator_amd import evaluacion as E
from music_generator_amd.graph import Input, Model
from music_generator_amd.layers import Conv2D, Flatten

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("flat,classes", [(True, 5), (True, 700), (False, 50)])
def test_frozen_head(flat, classes):
    """A head that is not trained leaves its weights and still passes the gradient of its input on."""
    gen = np.random.default_rng(0)
    x = gen.standard_normal((6, 2, 8, 4)).astype(np.float32)
    numbers = gen.integers(0, classes, (6,) if flat else (6, 2, 8))
    first = []
    for frozen in (False, True):
        M.clear_session()
        M.layers.set_init_seed(2)
        image = Input(shape=(2, 8, 4))
        t = Conv2D(32, (1, 1), padding="same")(image)
        head = E.SoftmaxDense(classes)
        model = Model(image, head(Flatten()(t) if flat else t))
        head.trainable = not frozen
        before = [v.numpy().copy() for v in (head.kernel, head.bias)]
        trunk, _ = E._split_head(model)
        model.bind_grads(0).zero_()
        features, _ = trunk.forward(torch.from_numpy(x).cuda(), save=True)
        first.append(head.loss(features, E.class_numbers_to_device(numbers)))
        E.fit_evaluator(model, x, numbers, 1, 3)
        moved = [bool((v.numpy() != w).any()) for v, w in zip((head.kernel, head.bias), before)]
        assert moved == [not frozen] * 2
    assert all(torch.equal(a, b) for a, b in zip(*first))
