"""The inputs that the operators are timed on are a function of the seed: two preparations
of one seed hold the same bits."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cases():
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


# (of 1000 tokens 30 drawn places repeat in a third of the rows)
@pytest.mark.parametrize("case", [
    {"op": "sample", "dtype": "bf16", "n": 512, "v": 1000, "t": 1.0, "k": 0, "p": 1.0, "m": 0.0, "mixed": False, "banned": 0.0,
     "flat": False},
    {"op": "sample", "dtype": "f32", "n": 64, "v": 5003, "t": 1.0, "k": 0, "p": 1.0, "m": 0.0, "mixed": True, "banned": 0.5,
     "flat": False},
    {"op": "norm_train", "dtype": "bf16", "n": 65, "h": 300, "residual": True, "offset": 0.0},
    {"op": "clip", "dtype": "f32", "layers": 2, "h": 33, "v": 1000, "out": "bf16", "reached": True},
], ids=lambda c: f"{c['op']}-{c['dtype']}")
def test_one_seed_gives_the_same_inputs(case):
    m = cases()

    def inputs(seed):
        return {k: v.detach().clone() for k, v in m.prepare(case, seed).items()
                if torch.is_tensor(v) and k != "out_flat"}   # (that one is written by the call)
    want = inputs(5)
    for _ in range(12):
        got = inputs(5)
        assert got.keys() == want.keys() and all(torch.equal(got[k], want[k]) for k in want)
    assert any(not torch.equal(a, b) for a, b in zip(inputs(6).values(), want.values()))
