"""examples/parallel_samples.py: samples that share pages give what each of them
gives alone."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("parallel_samples", os.path.join(ROOT, "examples", "parallel_samples.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_samples_share_pages(device, kind):
    ex = _example()
    model = ex.Model(3, device)
    g = torch.Generator(device="cpu").manual_seed(4)
    prompt = torch.randint(0, ex.WORDS, (150,), generator=g).to(device)
    noise = -torch.log(-torch.log(torch.rand(20, 4, ex.WORDS, generator=g).clamp(1e-9, 1 - 1e-7))).to(device)
    tokens, log_p, cache, active, moved = ex.generate(model, prompt, 4, 20, kind, noise, device)
    assert tokens.shape == (4, 20) and len(set(map(tuple, tokens.tolist()))) == 4
    # two pages of the prompt are shared by all four, the third was copied by each as it grew
    assert moved[1] == 2 + 4 and int(cache.refs[cache.refs > 0].sum()) == 4 * 3
    assert torch.equal(cache.refs[:moved[1]] > 0, torch.ones(moved[1], dtype=torch.bool, device=device))
    for row in range(4):
        # the same tokens alone: the prompt in one call, then one by one; the same codes, so only sums differ
        alone = torch.full_like(noise[:, :1], -1e9)
        alone[torch.arange(20), 0, tokens[row]] = 1e9
        again, want, single, _, _ = ex.generate(model, prompt, 1, 20, kind, alone, device)
        assert torch.equal(again[0], tokens[row])
        assert (log_p[row] - want[0]).abs().max() < 2e-4
        lengths = int(single.lengths[0])
        for entry in range(3):
            theirs, mine = int(cache.tables[active[row], entry]), int(single.tables[0, entry])
            assert torch.equal(cache.scales[:1, theirs], single.scales[:1, mine]) and lengths == 170


def test_command(device, capsys):
    _example().main(["--samples", "3", "--steps", "5", "--prompt", "70", "--kind", "e4m3"])
    assert "pages in use" in capsys.readouterr().out
