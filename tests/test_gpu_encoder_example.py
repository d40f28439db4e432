"""The example that trains an encoder, encodes a corpus and searches it, at a small size: the loss falls
and queries find their passages."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_encoder.py")


def test_train_encode_search(dev):
    spec = importlib.util.spec_from_file_location("train_encoder", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    args = ["--vocab", "3000", "--dim", "100", "--out", "96", "--passages", "3000", "--length", "40", "--steps", "60",
            "--batch", "256", "--nlist", "16", "--nprobe", "16"]
    got = example.main(args)
    assert got["last"] < 0.5 * got["first"], got
    # chance would be 10 of 3000
    assert got["hits"] > 0.3, got
    # every list is probed, so the index's answer is the exhaustive one but for float32 ties in the check
    assert got["recall"] > 0.999, got
