"""The example's generation from prompts of which some are empty."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generate_dna.py")
    spec = importlib.util.spec_from_file_location("generate_dna", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_an_empty_prompt_is_not_the_row_before_it(example):
    print("example: empty prompts", flush=True)
    torch.manual_seed(0)
    model = example.RecurrentLM(500).cuda()
    generator = example.Generator(model)
    gen = torch.Generator().manual_seed(1)
    chosen = []
    for lengths in ([40, 0, 3], [25, 0, 0], [0, 0, 0]):
        ids = torch.randint(0, 500, (sum(lengths),), generator=gen, dtype=torch.int32).cuda()
        offsets = torch.tensor([0] + lengths).cumsum(0).cuda()
        chosen.append(generator.generate(model, ids, offsets, 8)[1].tolist())
    assert chosen[0] == chosen[1] == chosen[2] and len(chosen[0]) == 8
