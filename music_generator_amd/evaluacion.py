"""The evaluator network and the Inception score computed from it: trainer/evaluacion.py:27-110 and
trainer/utils.py:65-76, inference side (the `evaluador.predict(gen_auds)` calls of
trainer/utils.py:98, 121).

The evaluator is a progressive family like the discriminator, but purely linear: 128-channel
convolutions without activations and a Dense(9, softmax) classifier head.  Its 128 -> 128
convolutions run on the library's general contraction kernel.  `load_evaluator` is the
download=False branch of evaluacion.py:114-166: fit the model of one resolution on (clips, one-hot
labels) with Adam (keras defaults) and categorical cross-entropy; the cloud download / upload of
the .h5 file is replaced by `Model.save` / `load_weights`.
"""
from __future__ import annotations

from typing import Dict, List, Optional

import numpy as np
import torch

from . import backend as K
from . import ops
from .graph import Input, Model
from .layers import Conv2D, Dense, Flatten


class SoftmaxDense(Dense):
    """Dense(units, activation='softmax') on a flattened input (evaluacion.py:97) or on every position of a feature map.
    With a tape the layer returns its LOGITS: the fitting loop pairs them with the fused softmax +
    cross-entropy kernel, whose logit gradient is what backward() receives.  Fitting on class numbers does not
    run this layer: `loss` takes its input and never stores the logits."""

    def forward(self, xs, save, act_alpha: float = 0.0):
        logits, saved = super().forward(xs, save, 0.0)
        if save:
            return logits, saved
        y = K.empty(logits.shape)
        ops.softmax_rows(logits.contiguous().view(-1, self.units), y.view(-1, self.units))
        return y, None

    def loss(self, features, labels, backward: bool = True):
        """(sum of the losses, hits, labelled rows, gradient of the mean loss with respect to `features` or None) of the
        head on `features` (..., cin) for class numbers `labels` (one per row of features; outside [0, units): no
        label), as 0-d device tensors.  With `backward` the gradients of the mean are added to the bound views of the
        head's variables.  The logits are never stored (ops.dense_xent_fwd / _bwd), unless they are no wider than the
        features beside them (the 9 classes of define_evaluator on 384 000 features): then storing them costs nothing."""
        x = features.reshape(-1, self.cin)
        n = x.shape[0]
        if labels.numel() != n:
            raise ops.MgxError("%s: %d class numbers for %d rows of features" % (self.name, labels.numel(), n))
        labelled = (labels >= 0) & (labels < self.units)
        count = labelled.sum().float()
        if self.units <= self.cin and features.dim() == 2:
            return self._loss_from_logits(x, labels, labelled, count, backward)
        w, b = self.kernel.value().view(self.cin, self.units), self.bias.value()
        loss, lse, hits = K.empty((n,)), K.empty((n,)), K.empty((n,), dtype=torch.int32)
        ops.dense_xent_fwd(x, w, b, labels, loss, lse, hits)
        dx = None
        if backward:
            dw = db = None                               # a frozen head passes the gradient on
            if self.trainable:
                if self.kernel.grad is None or self.bias.grad is None:
                    raise RuntimeError("gradient buffers of %s are not bound" % self.name)
                dw, db = self.kernel.grad.view(self.cin, self.units), self.bias.grad
            dx = torch.empty_like(x)
            ops.dense_xent_bwd(x, w, b, labels, lse, labelled.float() / count.clamp(min=1.0), dx, dw, db, accumulate=True)
            dx = dx.view(features.shape)
        return loss.sum(), hits.sum(), count, dx

    def _loss_from_logits(self, x, labels, labelled, count, backward):
        x = torch.where(labelled[:, None], x, torch.zeros_like(x))       # an unlabelled sample may hold anything
        logits, saved = super().forward([x], True)
        hot = torch.zeros_like(logits).scatter_(1, labels.long().clamp(0, self.units - 1)[:, None], 1.0)
        prob, rows, dlogits = K.empty(logits.shape), K.empty((x.shape[0],)), K.empty(logits.shape)
        ops.softmax_xent(logits.contiguous(), hot, prob, rows, dlogits)
        loss = torch.where(labelled, rows, torch.zeros_like(rows)).sum()
        hits = ((prob.argmax(dim=1) == labels) & labelled).sum()
        if not backward:
            return loss, hits, count, None
        # dlogits is the gradient of the mean over all rows
        dlogits = torch.where(labelled[:, None], dlogits * (x.shape[0] / count.clamp(min=1.0)), torch.zeros_like(dlogits))
        return loss, hits, count, super().backward(saved, dlogits, [True], [None], True)[0][0]


def _conv(t, ksize, **kw):
    return Conv2D(128, ksize, kernel_initializer="he_normal", **kw)(t)


def add_evaluator_block(old_model, n_input_layers=3):
    """evaluacion.py:27-65: a new 128-channel block at twice the resolution in front of the old
    model's layers from index `n_input_layers` on (so, as in the reference, the old model's input,
    its 1x1 feature convolution and its first 3x3 convolution are left out)."""
    in_shape = old_model.input.shape
    in_image = Input(shape=(in_shape[-3] * 2, in_shape[-2] * 2, in_shape[-1]))
    t = _conv(in_image, (1, 1), padding="same")
    for _ in range(2):                                   # convolution blocks 1 and 2
        t = _conv(t, (3, 3), padding="same")
        t = _conv(t, (3, 3), padding="same")
        t = _conv(t, (2, 2), padding="same")
    t = _conv(t, (3, 3), padding="same")                 # block 3 ends in the stride-2 reduction
    t = _conv(t, (3, 3), padding="same")
    t = _conv(t, (2, 2), strides=(2, 2), padding="valid")
    t = _conv(t, (1, 1), padding="same")
    final = None
    for layer in old_model.layers[n_input_layers:]:
        if isinstance(layer, Dense):
            final = layer(t)
        else:
            t = layer(t)
    return Model(in_image, final)


def define_evaluator(n_blocks, input_shape=(4, 750, 2)):
    """evaluacion.py:69-110: list of n_blocks models, one per resolution, sharing the old layers."""
    in_image = Input(shape=input_shape)
    t = _conv(in_image, (1, 1), padding="same")
    for _ in range(3):
        for ksize in ((3, 3), (4, 4), (3, 3)):
            t = _conv(t, ksize, padding="same")
    t = Flatten()(t)
    model_list = [Model(in_image, SoftmaxDense(9)(t))]
    for i in range(1, n_blocks):
        model_list.append(add_evaluator_block(model_list[i - 1]))
    return model_list


def calculate_inception_score(p_yx, eps=1e-16):
    """exp(mean_x KL(p(y|x) || p(y))) over a set of class-probability rows, trainer/utils.py:65-76
    (host arithmetic on the (n, 9) predictions)."""
    p_yx = np.asarray(p_yx.detach().cpu().numpy() if hasattr(p_yx, "detach") else p_yx, dtype=np.float64)
    p_y = p_yx.mean(axis=0, keepdims=True)
    kl = p_yx * (np.log(p_yx + eps) - np.log(p_y + eps))
    return float(np.exp(kl.sum(axis=1).mean()))


# evaluacion.py:130-157: batch size and epochs per resolution
FIT_TABLE = {4: (64, 10), 8: (32, 20), 16: (16, 30), 32: (8, 40), 64: (4, 50), 128: (2, 60), 256: (2, 70)}


def labels_to_device(y) -> torch.Tensor:
    """One-hot labels (n, classes) as a contiguous float32 device tensor."""
    t = y if isinstance(y, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(y, dtype=np.float32))
    return t.to(device=K.device(), dtype=torch.float32).contiguous()


def _class_numbers(y, model=None) -> bool:
    """Labels are class numbers (sparse categorical cross-entropy) rather than one-hot rows: an integer type, and not the
    shape of the model's output, which one-hot rows of any type have."""
    y = y if isinstance(y, torch.Tensor) else np.asarray(y)
    whole = not (y.is_floating_point() if isinstance(y, torch.Tensor) else np.issubdtype(y.dtype, np.floating))
    return whole and (model is None or tuple(y.shape[1:]) != tuple(model.output.shape[1:]))


def class_numbers_to_device(y) -> torch.Tensor:
    """Class numbers of any shape as a flat int32 device tensor; numbers that int32 does not hold become -1 (no label)."""
    t = y if isinstance(y, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(y))
    t = t.to(device=K.device(), dtype=torch.int64).reshape(-1)
    return torch.where((t >= 0) & (t < 2 ** 31), t, torch.full_like(t, -1)).to(torch.int32)


def _split_head(model):
    """(model of everything in front of the classifier head, head) for a model that ends in a SoftmaxDense."""
    node = model.output.node
    if not isinstance(node.layer, SoftmaxDense):
        raise ValueError("fitting on class numbers needs a model that ends in a SoftmaxDense")
    return Model(model.input, node.inputs[0]), node.layer


def evaluate(model, x, y, batch_size: int = 32) -> Dict[str, float]:
    """Mean categorical cross-entropy and accuracy over (x, y) - keras' evaluate / validation pass.  y: one-hot rows, or
    class numbers (one per sample or per position, negative: none), then the mean is over the labelled rows."""
    n = x.shape[0]
    if _class_numbers(y, model):
        trunk, head = _split_head(model)
        sums = torch.zeros((3,), dtype=torch.float64, device=K.device())
        for i in range(0, n, batch_size):
            features, _ = trunk.forward(model._to_device(x[i:i + batch_size]))
            loss, hits, count, _ = head.loss(features, class_numbers_to_device(y[i:i + batch_size]), backward=False)
            sums += torch.stack([loss.double(), hits.double(), count.double()])
        loss, hits, count = sums.tolist()
        return {"loss": loss / max(count, 1.0), "accuracy": hits / max(count, 1.0)}
    loss, hits = 0.0, 0
    for i in range(0, n, batch_size):
        xb = model._to_device(x[i:i + batch_size])
        yb = labels_to_device(y[i:i + batch_size])
        logits, _ = model.forward(xb, save=True)          # with a tape the head returns logits
        prob, rows = K.empty(logits.shape), K.empty((logits.shape[0],))
        ops.softmax_xent(logits.contiguous(), yb, prob, rows, None)
        loss += float(rows.sum())
        hits += int((prob.argmax(dim=1) == yb.argmax(dim=1)).sum())
    return {"loss": loss / n, "accuracy": hits / n}


def fit_evaluator(model, x, y, epochs: int, batch_size: int, optimizer=None, validation_data=None,
                  shuffle_seed: int = 0, verbose: int = 0) -> Dict[str, List[float]]:
    """model.compile(optimizer="Adam", loss='categorical_crossentropy', metrics=["accuracy"]) +
    model.fit(X, y, epochs, batch_size, validation_data) of evaluacion.py:160-161.  Returns the
    history: per epoch the sample-weighted mean of the batch losses / accuracies (and val_*).

    y as an integer array that has not the shape of one-hot rows holds class numbers (keras' sparse categorical cross-entropy): one per
    sample, or one per position for a head without a Flatten in front; negative numbers are positions without a label, and
    a batch's loss is the mean over its labelled ones.  The logits of that form are never stored, so that it is the one for
    many classes or many positions; backend.TAPE8 keeps the rest of the tape in 8 bits."""
    from .models import Adam
    opt = optimizer or Adam()                              # keras defaults: 1e-3, 0.9, 0.999, 1e-7
    n = x.shape[0]
    rng = np.random.default_rng(shuffle_seed)
    hist: Dict[str, List[float]] = {"loss": [], "accuracy": []}
    numbers = _class_numbers(y, model)
    if numbers:
        trunk, head = _split_head(model)
        y = np.ascontiguousarray(y.cpu().numpy() if isinstance(y, torch.Tensor) else y)
        if y.shape[0] != n:
            raise ValueError("one row of class numbers per sample expected")
    else:
        y = np.ascontiguousarray(y, dtype=np.float32)
    for epoch in range(epochs):
        order = rng.permutation(n)
        loss_sum = torch.zeros((), dtype=torch.float32, device=K.device())
        hits = torch.zeros((), dtype=torch.int64, device=K.device())
        counted = torch.zeros((), dtype=torch.float64, device=K.device())
        for i in range(0, n, batch_size):
            idx = order[i:i + batch_size]
            if numbers:
                model.bind_grads(0).zero_()
                features, tape = trunk.forward(model._to_device(x[idx]), save=True)
                loss, right, count, dx = head.loss(features, class_numbers_to_device(y[idx]))
                trunk.backward(tape, dx, need_input_grad=False)
                opt.apply_model_gradients(model)
                loss_sum += loss
                hits += right
                counted += count
                continue
            xb, yb = model._to_device(x[idx]), labels_to_device(y[idx])
            flat = model.bind_grads(0)
            flat.zero_()
            logits, tape = model.forward(xb, save=True)
            prob, rows, dlogits = K.empty(logits.shape), K.empty((logits.shape[0],)), K.empty(logits.shape)
            ops.softmax_xent(logits.contiguous(), yb, prob, rows, dlogits)
            model.backward(tape, dlogits, need_input_grad=False)
            opt.apply_model_gradients(model)
            loss_sum += rows.sum()
            hits += (prob.argmax(dim=1) == yb.argmax(dim=1)).sum()
        total = max(float(counted), 1.0) if numbers else n
        hist["loss"].append(float(loss_sum) / total)
        hist["accuracy"].append(int(hits) / total)
        if validation_data is not None:
            val = evaluate(model, validation_data[0], validation_data[1], batch_size)
            hist.setdefault("val_loss", []).append(val["loss"])
            hist.setdefault("val_accuracy", []).append(val["accuracy"])
        if verbose:
            print("epoch %d/%d " % (epoch + 1, epochs) + " ".join("%s=%.4f" % (k, v[-1]) for k, v in hist.items()))
    return hist


def load_evaluator(dimension, train_dataset, epochs: Optional[int] = None, n_blocks: int = 7, verbose: int = 0):
    """evaluacion.py:114-166 with download=False: build the family, pick the model of `dimension`
    (H, W), fit it on train_dataset = (X, one-hot y) with the batch size / epochs of the
    reference's table, validating on the training set as the reference does.  Returns the model
    (history in `model.fit_history`)."""
    batch_size, table_epochs = FIT_TABLE[int(dimension[0])]
    stage = int(dimension[0]).bit_length() - 3            # 4 -> 0, 8 -> 1, ...
    model = define_evaluator(max(n_blocks, stage + 1))[stage]
    x, y = train_dataset
    model.fit_history = fit_evaluator(model, x, y, table_epochs if epochs is None else epochs, batch_size,
                                      validation_data=(x, y), verbose=verbose)
    return model
