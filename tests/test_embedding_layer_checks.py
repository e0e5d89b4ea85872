"""EmbeddingEncoder's norm, dropout and products are checked before a device is
touched."""
import numpy as np
import pytest

from mlrs_amd.embedding import EmbeddingEncoder


@pytest.mark.parametrize("kw,words", [
    (dict(norm_groups=3), "norm_groups should divide"), (dict(norm_groups=0), "norm_groups should divide"),
    (dict(dropout=1.0), "dropout should be in"), (dict(dropout=-0.1), "dropout should be in"),
    (dict(dropout=float("nan")), "dropout should be in"), (dict(products="int8"), "products should be"),
])
def test_parameters(kw, words):
    with pytest.raises(ValueError, match=words):
        EmbeddingEncoder(hidden=(16, 32), **kw).fit(np.zeros((3, 2)), np.zeros(3))
