"""Training the rows that the engine searches: ``EmbeddingEncoder`` learns a
dense encoder whose outputs separate given classes, for ``NearestNeighbors``,
``KNeighborsClassifier`` or ``KMeans`` over ``transform(X)``.  No counterpart in
the reference.

The network is layers ``drop(act(x w^T + b))``, a layer as wide as its input
adding it (``+ x``), a last linear layer to ``n_components`` columns, and a class
head ``h w^T + b`` under a softmax.  With ``norm_groups`` a layer is
``drop(act(group_norm(x w^T + b)))``; with ``products="fp8"`` the products of all
layers but the head are those of 8-bit values, forwards and backwards.  Every
product, norm, activation and gradient, dropout, the loss over the classes and the
optimizer's step are the library's kernels (``prims.linear``, ``linear_grad``,
``group_norm``, ``group_norm_grad``, ``dropout``, ``fp8_weight``, ``linear_fp8``,
``linear_fp8_grad``, ``softmax_xent``, ``softmax_xent_grad``, ``clip_scale``,
``adamw_step``): the logits of a batch and dropout's masks are never in memory, and
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
    the optimizer's moments.  ``norm_groups``: None, or the groups of a group norm
    (1: layer norm) between a hidden layer's product and its activation, a divisor of
    every hidden width.  ``dropout`` in [0, 1) is a hidden layer's, in ``fit`` alone.
    ``products``: "native", or "fp8" for 8-bit floating point with a scale for each
    128 elements; the weights are kept in ``dtype`` and made into codes every step,
    and once for the fitted encoder.  A step takes ``batch_size`` rows; ``epochs`` is
    the number of passes over the rows.  ``random_state=None`` is seed 0.

    After ``fit``: ``classes_``, ``loss_curve_`` (the mean loss of each epoch),
    ``n_features_in_``.  Steps whose gradients are not finite are skipped (with
    ``max_norm`` or float16), and a warning tells how many they were.
    """

    def __init__(self, n_components=64, hidden=(256,), activation="gelu", epochs=10, batch_size=1024,
                 learning_rate=1e-3, weight_decay=0.01, max_norm=1.0, dtype="float32", state_bits=32,
                 random_state=None, output_type="input", norm_groups=None, dropout=0.0, products="native"):
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
        self.norm_groups = norm_groups
        self.dropout = dropout
        self.products = products

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
        if self.norm_groups is not None:
            if int(self.norm_groups) < 1 or any(w % int(self.norm_groups) for w in widths[:-1]):
                raise ValueError("norm_groups should divide every hidden width %r, got %r"
                                 % (widths[:-1], self.norm_groups))
        if not 0.0 <= float(self.dropout) < 1.0:
            raise ValueError("dropout should be in [0, 1), got %r" % (self.dropout,))
        if self.products not in ("native", "fp8"):
            raise ValueError("products should be 'native' or 'fp8', got %r" % (self.products,))
        return widths

    def _init_params(self, d, widths, classes, device, gen):
        """Weights of variance 1 / inputs, biases zero, the norms' weights one: [w, b]
        of every layer, of a hidden one with a norm [w, b, norm's weight, its bias];
        the class head last."""
        out = []
        dtype = _DTYPES[self.dtype]
        for i, wide in enumerate(widths + [classes]):
            w = torch.empty(wide, d, dtype=torch.float32, device=device).normal_(0.0, d ** -0.5, generator=gen)
            out += [w.to(dtype), torch.zeros(wide, dtype=dtype, device=device)]
            if self.norm_groups is not None and i < len(widths) - 1:
                out += [torch.ones(wide, dtype=dtype, device=device), torch.zeros(wide, dtype=dtype, device=device)]
            d = wide
        return out

    def _layers(self):
        """(w, b, norm's weight and bias or None, activation, whether the input is
        added) of every layer but the head; the last has neither norm, activation
        nor sum."""
        out, at = [], 0
        each = 2 if self.norm_groups is None else 4
        while at < len(self._params) - 4:
            w, b = self._params[at:at + 2]
            norm = None if each == 2 else self._params[at + 2:at + 4]
            out.append((w, b, norm, self.activation, w.shape[0] == w.shape[1]))
            at += each
        w, b = self._params[at:at + 2]
        return out + [(w, b, None, "none", False)]

    def _codes(self, backward):
        """The layers' weights in 8 bits, None for each with native products."""
        return [prims.fp8_weight(layer[0], backward=backward) if self.products == "fp8" else None
                for layer in self._layers()]

    @staticmethod
    def _product(x, w, w8, **kw):
        return prims.linear(x, w, **kw) if w8 is None else prims.linear_fp8(x, w8, **kw)

    def _encode(self, x):
        layers = self._layers()
        # the fitted weights', or, of a fit that was interrupted, those of its weights
        codes = self._weight_codes if self.products == "fp8" else None
        if codes is None:
            codes = self._codes(backward=False)
        for (w, b, norm, act, skip), w8 in zip(layers, codes):
            if norm is None:
                x = self._product(x, w, w8, bias=b, activation=act, residual=x if skip else None)
                continue
            y = prims.group_norm(self._product(x, w, w8, bias=b), int(self.norm_groups), weight=norm[0], bias=norm[1],
                                 activation=act)
            x = y.add_(x) if skip else y
        return x

    def _loss_and_grads(self, x, target, weight, seed=0, step=0):
        """The rows' losses, and the gradients of sum(weight * loss) in the order
        of the parameters.  `seed` and `step` decide dropout's masks."""
        layers, codes = self._layers(), self._codes(backward=True)
        p = float(self.dropout)
        kept = []
        for i, ((w, b, norm, act, skip), w8) in enumerate(zip(layers, codes)):
            hidden = i < len(layers) - 1
            drop = dict(p=p if hidden else 0.0, seed=seed, offset=step * len(layers) + i)
            # where the input is added, dropout comes with the sum, after the layer
            late = hidden and p > 0.0 and (skip or norm is None)
            if norm is None:
                y, z = self._product(x, w, w8, bias=b, activation=act, keep_preact=True,
                                     residual=x if skip and not late else None)
                stats = None
            else:
                z = self._product(x, w, w8, bias=b)
                within = {} if late else drop
                y, *stats = prims.group_norm(z, int(self.norm_groups), weight=norm[0], bias=norm[1], activation=act,
                                             keep_stats=True, **within)
                if skip and not late:
                    y += x
            if late:
                y = prims.dropout(y, residual=x if skip else None, **drop)
            kept.append((x, z, stats, drop, late))
            x = y
        head, bias = self._params[-2:]
        loss, lse = prims.softmax_xent(x, head, target, bias=bias)
        dx, dw, db = prims.softmax_xent_grad(x, head, target, lse, weight, bias=bias)
        grads = [dw, db]
        for i in range(len(layers) - 1, -1, -1):
            w, b, norm, act, skip = layers[i]
            x, z, stats, drop, late = kept[i]
            dy = dx
            inner = prims.dropout(dy, **drop) if late else dy
            more = []
            if norm is not None:
                inner, *more = prims.group_norm_grad(inner, z, *stats, weight=norm[0], bias=norm[1], activation=act,
                                                     **({} if late else drop))
                z, act = None, "none"
            if codes[i] is None:
                dx, dw, db = prims.linear_grad(inner, x, w, preact=z, activation=act, need_dx=i > 0)
            else:
                dx, dw, db = prims.linear_fp8_grad(inner, x, codes[i], preact=z, activation=act, need_dx=i > 0)
            if skip and i > 0:
                dx += dy
            grads = [dw, db] + more + grads
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
        classes, codes = np.unique(labels, return_inverse=True)
        target = torch.from_numpy(np.ascontiguousarray(codes.reshape(-1), dtype=np.int64)).to(x.device)
        n, d = x.shape
        seed = 0 if self.random_state is None else int(self.random_state)
        gen = torch.Generator(device=x.device)
        gen.manual_seed(seed)
        params = self._init_params(d, widths, len(classes), x.device, gen)
        optimizer = AdamW(params, lr=float(self.learning_rate), weight_decay=float(self.weight_decay),
                          max_norm=self.max_norm, state_bits=self.state_bits, seed=seed)
        # from here on nothing of an earlier fit is left
        self.classes_, self.n_features_in_, self._params, self._weight_codes = classes, d, params, None
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
                loss, grads = self._loss_and_grads(x[rows], target[rows], weight, seed, steps)
                norm = optimizer.step(grads)
                steps += 1
                if norm is not None:
                    norms.append(norm)
                total += loss.sum()
            self.loss_curve_.append(total / n)
            if norms:
                skipped.append((~torch.cat(norms).isfinite()).sum())
                norms = []
        if self.products == "fp8":
            self._weight_codes = self._codes(backward=False)
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
