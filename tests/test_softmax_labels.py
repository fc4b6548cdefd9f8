"""Labels that SoftmaxClassifier can be trained on and those that its files hold."""
import datetime
import fractions
import os

import numpy as np
import pytest

from image_classification_amd import SoftmaxClassifier
from test_softmax_classifier import LearnChecker, blobs


def trained(labels, x):
    c = SoftmaxClassifier(epochs=1, backend=LearnChecker())
    c.train(x, labels)
    return c


@pytest.mark.parametrize("of", [int, float, str, bool, lambda i: bytes([65 + i]), np.int64, np.float32],
                         ids=["int", "float", "str", "bool", "bytes", "int64", "float32"])
def test_labels_survive_the_file(of, tmp_path):
    x, y = blobs(60, 3, 5, 0)
    c = trained([of(int(i)) for i in y], x)
    c.save_to_file(str(tmp_path / "c"))
    again = SoftmaxClassifier.load_from_file(str(tmp_path / "c"), backend=LearnChecker())
    assert again.labels_map == c.labels_map and (again.test(x) == c.test(x)).all()


@pytest.mark.parametrize("of", [lambda i: 10 ** 30 + i, lambda i: fractions.Fraction(i, 3),
                                lambda i: datetime.date(2020, 1, 1 + i)], ids=["big", "fraction", "date"])
def test_labels_that_only_a_pickle_could_hold_are_refused_by_the_file(of, tmp_path):
    x, y = blobs(60, 3, 5, 0)
    c = trained([of(int(i)) for i in y], x)
    assert c.test(x[:1])[0] in c.labels_map
    path = tmp_path / "c"
    path.write_bytes(b"an older file")
    with pytest.raises(ValueError, match="pickl"):
        c.save_to_file(str(path))
    assert path.read_bytes() == b"an older file" and os.listdir(tmp_path) == ["c"]
