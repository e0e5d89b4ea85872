"""Training the rows that the engine searches: ``EmbeddingEncoder`` learns a
dense encoder whose outputs separate given classes, for ``NearestNeighbors``,
``KNeighborsClassifier`` or ``KMeans`` over ``transform(X)``.  No counterpart in
the reference.

The network is layers ``act(x w^T + b)``, a layer as wide as its input adding
it (``+ x``), a last linear layer to ``n_components`` columns, and a class head
``h w^T + b`` under a softmax.  Every product, its activation and its gradient,
the loss over the classes and the optimizer's step are the library's kernels
(``prims.linear``, ``linear_grad``, ``softmax_xent``, ``softmax_xent_grad``,
``clip_scale``, ``adamw_step``): the logits of a batch are never in memory, and
a step reads nothing back.
"""
import warnings

import numpy as np
import torch

from . import prims
from .neighbors import _as_device_matrix, _check_finite

_LOGITS = 1 << 26  # that predict holds at a time
_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


class AdamW:
    """The optimizer state of a list of float32, float16 or bfloat16 tensors:
    their moments in 32 or in 8 bits, and float32 masters of 16-bit parameters.

    ``step(grads)`` takes one step in place; with ``max_norm`` the gradients are
    clipped to that norm first, and a step whose norm is not finite changes
    nothing but the count of steps; float16 parameters, whose gradients may leave
    the type's range, have that without a ``max_norm`` too.  Tensors of one
    dimension do not decay."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_norm=None, state_bits=32,
                 seed=0):
        if state_bits not in (32, 8):
            raise ValueError("state_bits should be 32 or 8, got %r" % (state_bits,))
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        self.lr, self.betas, self.eps, self.max_norm, self.seed = lr, betas, eps, max_norm, int(seed)
        self.decays = [weight_decay if p.dim() > 1 else 0.0 for p in self.params]
        half = [p.dtype != torch.float32 for p in self.params]
        if any(half) != all(half):
            raise ValueError("float32 and 16-bit parameters cannot share an optimizer")
        self.masters = [p.float() for p in self.params] if half[0] else None
        self.overflows = any(p.dtype == torch.float16 for p in self.params)
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg = [torch.zeros_like(p, dtype=kind) for p in self.params]
        self.exp_avg_sq = [torch.zeros_like(p, dtype=kind) for p in self.params]
        self.avg_scales = self.avg_sq_scales = None
        if state_bits == 8:
            self.avg_scales, self.avg_sq_scales = (
                [torch.zeros(-(-p.numel() // prims.STATE_BLOCK), dtype=torch.float32, device=p.device)
                 for p in self.params] for _ in range(2))
        self.steps = 0

    def step(self, grads):
        """One step; returns the gradients' norm (a device tensor) with
        ``max_norm`` or float16 parameters, else None."""
        norm = scale = None
        if self.max_norm is not None or self.overflows:
            norm, scale = prims.clip_scale(grads, float("inf") if self.max_norm is None else self.max_norm)
        self.steps += 1
        prims.adamw_step(self.params, grads, self.exp_avg, self.exp_avg_sq, step=self.steps, lr=self.lr,
                         betas=self.betas, eps=self.eps, weight_decay=self.decays, masters=self.masters,
                         avg_scales=self.avg_scales, avg_sq_scales=self.avg_sq_scales, scale=scale,
                         seed=(self.seed + self.steps * 0x85EBCA6B) & 0xFFFFFFFF)
        return norm


class EmbeddingEncoder:
    """A dense encoder trained to tell classes apart.

    ``hidden`` are the widths of the hidden layers, ``n_components`` that of the
    embedding; ``activation`` one of ``prims.ACTIVATIONS``; ``dtype`` the
    element type of the parameters and the products ("float32", "float16" or
    "bfloat16", the 16-bit types with float32 masters); ``state_bits`` that of
    the optimizer's moments.  A step takes ``batch_size`` rows; ``epochs`` is
    the number of passes over the rows.  ``random_state=None`` is seed 0.

    After ``fit``: ``classes_``, ``loss_curve_`` (the mean loss of each epoch),
    ``n_features_in_``.  Steps whose gradients are not finite are skipped (with
    ``max_norm`` or float16), and a warning tells how many they were.
    """

    def __init__(self, n_components=64, hidden=(256,), activation="gelu", epochs=10, batch_size=1024,
                 learning_rate=1e-3, weight_decay=0.01, max_norm=1.0, dtype="float32", state_bits=32,
                 random_state=None, output_type="input"):
        self.n_components = n_components
        self.hidden = hidden
        self.activation = activation
        self.epochs = epochs
        self.batch_size = batch_size
        self.learning_rate = learning_rate
        self.weight_decay = weight_decay
        self.max_norm = max_norm
        self.dtype = dtype
        self.state_bits = state_bits
        self.random_state = random_state
        self.output_type = output_type

    def _validate(self):
        if self.dtype not in _DTYPES:
            raise ValueError("dtype should be one of %s, got %r" % (sorted(_DTYPES), self.dtype))
        if self.activation not in prims.ACTIVATIONS:
            raise ValueError("activation should be one of %s, got %r" % (sorted(prims.ACTIVATIONS), self.activation))
        widths = [int(w) for w in self.hidden] + [int(self.n_components)]
        if min(widths) < 1:
            raise ValueError("layer widths should be > 0, got %r" % (widths,))
        for name in ("epochs", "batch_size"):
            if int(getattr(self, name)) < 1:
                raise ValueError("%s should be > 0, got %r" % (name, getattr(self, name)))
        return widths

    def _init_params(self, d, widths, classes, device, gen):
        """Weights of variance 1 / inputs, biases zero: [w, b] of every layer,
        the class head last."""
        out = []
        for wide in widths + [classes]:
            w = torch.empty(wide, d, dtype=torch.float32, device=device).normal_(0.0, d ** -0.5, generator=gen)
            out += [w.to(_DTYPES[self.dtype]), torch.zeros(wide, dtype=_DTYPES[self.dtype], device=device)]
            d = wide
        return out

    def _layers(self):
        """(w, b, activation, whether the input is added) of every layer but the head."""
        pairs = list(zip(self._params[0:-2:2], self._params[1:-2:2]))
        last = len(pairs) - 1
        return [(w, b, self.activation if i < last else "none", i < last and w.shape[0] == w.shape[1])
                for i, (w, b) in enumerate(pairs)]

    def _encode(self, x):
        for w, b, act, skip in self._layers():
            x = prims.linear(x, w, bias=b, activation=act, residual=x if skip else None)
        return x

    def _loss_and_grads(self, x, target, weight):
        """The rows' losses, and the gradients of sum(weight * loss) in the order
        of the parameters."""
        layers = self._layers()
        kept = []
        for w, b, act, skip in layers:
            y, z = prims.linear(x, w, bias=b, activation=act, residual=x if skip else None, keep_preact=True)
            kept.append((x, z))
            x = y
        head, bias = self._params[-2:]
        loss, lse = prims.softmax_xent(x, head, target, bias=bias)
        dx, dw, db = prims.softmax_xent_grad(x, head, target, lse, weight, bias=bias)
        grads = [dw, db]
        for i in range(len(layers) - 1, -1, -1):
            w, b, act, skip = layers[i]
            x, z = kept[i]
            dy = dx
            dx, dw, db = prims.linear_grad(dy, x, w, preact=z, activation=act, need_dx=i > 0)
            if skip and i > 0:
                dx += dy
            grads = [dw, db] + grads
        return loss, grads

    def fit(self, X, y):
        widths = self._validate()
        x, _ = _as_device_matrix(X)
        x = x.to(_DTYPES[self.dtype])
        _check_finite(x)  # as the layers read it: 65520 is no float16
        labels = y.cpu().numpy() if isinstance(y, torch.Tensor) else np.asarray(y)
        if labels.shape != (x.shape[0],):
            raise ValueError("y has shape %s, expected (%d,)" % (labels.shape, x.shape[0]))
        if x.shape[0] == 0 or x.shape[1] == 0:
            raise ValueError("Found array with shape %s: at least one row and one feature are required"
                             % (tuple(x.shape),))
        self.classes_, codes = np.unique(labels, return_inverse=True)
        target = torch.from_numpy(np.ascontiguousarray(codes.reshape(-1), dtype=np.int64)).to(x.device)
        n, d = x.shape
        seed = 0 if self.random_state is None else int(self.random_state)
        gen = torch.Generator(device=x.device)
        gen.manual_seed(seed)
        self.n_features_in_ = d
        self._params = self._init_params(d, widths, len(self.classes_), x.device, gen)
        optimizer = AdamW(self._params, lr=float(self.learning_rate), weight_decay=float(self.weight_decay),
                          max_norm=self.max_norm, state_bits=self.state_bits, seed=seed)
        # half precision's gradients are scaled into its range; AdamW's step does
        # not depend on a gradient's scale but through eps, which is scaled too
        up = 1024.0 if self.dtype == "float16" else 1.0
        if up != 1.0:
            optimizer.eps *= up
            if optimizer.max_norm is not None:
                optimizer.max_norm *= up
        self.loss_curve_, norms, skipped, steps = [], [], [], 0
        for _ in range(int(self.epochs)):
            order = torch.randperm(n, device=x.device, generator=gen)
            total = torch.zeros((), dtype=torch.float32, device=x.device)
            for start in range(0, n, int(self.batch_size)):
                rows = order[start:start + int(self.batch_size)]
                weight = torch.full((len(rows),), up / len(rows), dtype=torch.float32, device=x.device)
                loss, grads = self._loss_and_grads(x[rows], target[rows], weight)
                norm = optimizer.step(grads)
                steps += 1
                if norm is not None:
                    norms.append(norm)
                total += loss.sum()
            self.loss_curve_.append(total / n)
            if norms:
                skipped.append((~torch.cat(norms).isfinite()).sum())
                norms = []
        self.loss_curve_ = torch.stack(self.loss_curve_).cpu().tolist()
        skipped = int(sum(skipped))
        if skipped:
            warnings.warn("%d of %d steps were skipped: their gradients are not finite in %s (scale the features down, "
                          "or use another dtype)" % (skipped, steps, self.dtype), RuntimeWarning, stacklevel=2)
        return self

    def _check_fitted(self):
        if not hasattr(self, "_params"):
            raise ValueError("This EmbeddingEncoder instance is not fitted yet.")

    def _rows(self, X):
        self._check_fitted()
        x, was_numpy = _as_device_matrix(X, device=self._params[0].device)
        if x.shape[1] != self.n_features_in_:
            raise ValueError("X has %d features, but EmbeddingEncoder is expecting %d features as input"
                             % (x.shape[1], self.n_features_in_))
        x = x.to(_DTYPES[self.dtype])
        _check_finite(x)
        return x, was_numpy

    def transform(self, X):
        """The embedding of every row, float32 (n, n_components)."""
        x, was_numpy = self._rows(X)
        h = self._encode(x).float()
        return h.cpu().numpy() if was_numpy else h

    def fit_transform(self, X, y):
        return self.fit(X, y).transform(X)

    def predict(self, X):
        """The class the head gives each row, as ``fit`` was given it: a NumPy
        array, whatever holds the rows.  The logits are float32, as in the loss:
        rounded to a 16-bit type, near classes would tie."""
        x, _ = self._rows(X)
        h = self._encode(x)
        head, bias = (p.float() for p in self._params[-2:])
        code = torch.empty(len(h), dtype=torch.int64, device=h.device)
        rows = max(1, _LOGITS // len(head))
        for i in range(0, len(h), rows):
            code[i:i + rows] = prims.linear(h[i:i + rows].float(), head, bias=bias).argmax(1)
        return self.classes_.take(code.cpu().numpy())

    def score(self, X, y):
        """The mean cross entropy of the rows, lower is better."""
        x, _ = self._rows(X)
        labels = y.cpu().numpy() if isinstance(y, torch.Tensor) else np.asarray(y)
        place = np.searchsorted(self.classes_, labels)
        if np.any(place == len(self.classes_)) or np.any(self.classes_[np.minimum(place, len(self.classes_) - 1)]
                                                         != labels):
            raise ValueError("y holds classes that fit has not seen")
        target = torch.from_numpy(np.ascontiguousarray(place, dtype=np.int64)).to(x.device)
        loss, _ = prims.softmax_xent(self._encode(x), self._params[-2], target, bias=self._params[-1])
        return float(loss.mean())
