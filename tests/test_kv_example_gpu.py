"""examples/paged_decode.py: a step at a time gives what one step over the
whole sequences gives, up to the 8-bit codes (a page's scale grows token by
token there and is known at once here) and fp16."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_decode.py"


def _example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("page_size", [16, 64])
def test_steps_against_one_step(page_size):
    ex = _example()
    model = ex.Decoder(layers=2)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (37, 5, 0, 130, 64)]
    out, last = ex.generate(model, prompts, 20, page_size)
    assert out.shape == (5, 20)
    again, batch = ex.last_logits(model, prompts, out, page_size)
    live = [0, 1, 3, 4]
    # Codes are half a step of 1/127 of a page's largest off, once more for
    # each time its scale grew: about 1% of a value, which softmax and sums over
    # keys average; the logits' own size is 1.
    err = (again[live] - last[live]).float()
    assert (err.norm() / last[live].float().norm()).item() < 0.05
    assert batch.held.tolist() == [57, 25, 0, 150, 84]


def test_pages_run_out_raises():
    ex = _example()
    model = ex.Decoder(layers=1)

    class Short(ex.Batch):
        def __init__(self, model, places, pages, *args):
            super().__init__(model, places, pages, *args)
            self.free_count = torch.tensor([3], dtype=torch.int32, device="cuda")

    ex.Batch = Short
    with pytest.raises(RuntimeError, match="pages were missing"):
        ex.generate(model, [list(range(40)), list(range(30))], 2)
