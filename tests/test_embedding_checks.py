"""EmbeddingEncoder's parameters are checked before a device is touched."""
import numpy as np
import pytest

from mlrs_amd.embedding import EmbeddingEncoder


@pytest.mark.parametrize("kw,words", [
    (dict(dtype="float64"), "dtype should be one of"), (dict(activation="tanh"), "activation should be one of"),
    (dict(hidden=(8, 0)), "layer widths"), (dict(n_components=0), "layer widths"), (dict(epochs=0), "epochs"),
    (dict(batch_size=0), "batch_size"),
])
def test_parameters(kw, words):
    with pytest.raises(ValueError, match=words):
        EmbeddingEncoder(**kw).fit(np.zeros((3, 2)), np.zeros(3))


def test_not_fitted():
    with pytest.raises(ValueError, match="not fitted"):
        EmbeddingEncoder().transform(np.zeros((3, 2)))
