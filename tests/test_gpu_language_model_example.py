"""The training example: repeated passages against a dictionary of them, and a loss that falls."""
import importlib.util
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_on_documents.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_on_documents", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("passage", [1, 4, 20])
def test_repeated_passages_are_those_that_a_dictionary_finds(example, passage):
    rng = np.random.RandomState(passage)
    text = rng.randint(0, 4, 3000).astype(np.uint16)
    text[2000:2200] = text[100:300]
    text[::501] = 0xFFFF
    want, seen = [], set()
    for i in range(text.size):
        key = tuple(text[i:i + passage]) if i + passage <= text.size else i
        want.append(key in seen)
        seen.add(key)
    got = example.repeated(torch.from_numpy(text.view(np.int16)).cuda(), passage)
    assert got.tolist() == want


def test_training_lowers_the_loss(example):
    lines = []
    losses, share = example.train(tokens=30000, steps=12, length=2048, say=lines.append)
    assert len(losses) == 12 and len(lines) == 13
    assert all(np.isfinite(losses)) and 0 < share < 0.5
    assert abs(losses[0] - np.log(50257)) < 2 and np.mean(losses[-3:]) < np.mean(losses[:3]) - 0.5
