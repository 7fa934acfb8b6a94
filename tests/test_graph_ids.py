"""Categorical codes on their way into a graph: convert_to_graph(X, y, ids)."""
import numpy as np
import pandas as pd
import pytest
import torch


def test_codes_travel_with_the_graph():
    from gat_amd.data import convert_to_graph
    rng = np.random.default_rng(0)
    X, y = rng.random((40, 3)), rng.integers(0, 2, 40)
    assert convert_to_graph(X, y).ids is None
    codes = rng.integers(-1, 9, (40, 2)).astype(np.int32)
    for ids in (codes, pd.DataFrame(codes), codes[:, 0], pd.Series(codes[:, 0])):
        d = convert_to_graph(X, y, ids)
        assert d.ids.dtype == torch.int64 and np.array_equal(d.ids.numpy(), np.asarray(ids))
        assert torch.equal(d.to("cpu").ids, d.ids)
    for bad in (codes[:39], codes.astype(float), codes[None], np.int64(3)):
        with pytest.raises(ValueError, match="ids"):
            convert_to_graph(X, y, bad)
