"""Host side of the training step's prompts: what it takes, what it refuses, and what a refused call leaves as it was."""

from __future__ import annotations

import pytest
import torch

from fp8_b200.train import GraphedTrainStep


class _Step(GraphedTrainStep):
    """The step's inputs alone: its body does nothing."""

    def __init__(self, prompts: bool):
        self.static_batch, self.static_t = torch.zeros(2, 3, 4, 4), torch.zeros(2, dtype=torch.int64)
        self.static_eps, self.graph, self.ran = torch.zeros(2, 3, 4, 4), None, 0
        self.static_prompt = (torch.zeros(2, 5, dtype=torch.int64), torch.full((2,), 5, dtype=torch.int32)) if prompts else ()

    def _body(self):
        self.ran += 1


IMAGES, IDS, LENGTHS = torch.ones(2, 3, 4, 4), torch.arange(10).view(2, 5), torch.tensor([3, 1])


def test_prompts_are_copied_in():
    s = _Step(True)
    s.step(IMAGES, prompt_ids=IDS, prompt_lengths=LENGTHS)
    assert torch.equal(s.static_prompt[0], IDS) and s.static_prompt[1].tolist() == [3, 1] and s.ran == 1
    s.step()  # the same again
    assert torch.equal(s.static_prompt[0], IDS) and s.static_prompt[1].tolist() == [3, 1] and s.ran == 2
    s.step(IMAGES, prompt_ids=IDS + 1)  # whole prompts, not the last step's lengths
    assert torch.equal(s.static_prompt[0], IDS + 1) and s.static_prompt[1].tolist() == [5, 5]


@pytest.mark.parametrize("prompts,given,word", [
    (False, {"prompt_ids": IDS}, "without prompt_vocab"),
    (False, {"prompt_lengths": LENGTHS}, "without prompt_vocab"),
    (True, {}, "need their prompt_ids"),
    (True, {"prompt_lengths": LENGTHS}, "need their prompt_ids"),
    (True, {"prompt_ids": IDS[:1]}, "prompt_ids must be"),
    (True, {"prompt_ids": IDS[:, :4]}, "prompt_ids must be"),
    (True, {"prompt_ids": IDS[0]}, "prompt_ids must be"),
    (True, {"prompt_ids": IDS, "prompt_lengths": LENGTHS[:1]}, "prompt_lengths must be"),
    (True, {"prompt_ids": IDS, "prompt_lengths": torch.tensor(3)}, "prompt_lengths must be")])
def test_refusals(prompts, given, word):
    s = _Step(prompts)
    with pytest.raises(RuntimeError, match=word):
        s.step(IMAGES, **given)
    assert s.ran == 0 and torch.count_nonzero(s.static_batch) == 0
    s.step(IMAGES, **({"prompt_ids": IDS} if prompts else {}))
    assert s.ran == 1


def test_lengths_alone_are_refused_without_images_too():
    with pytest.raises(RuntimeError, match="need their prompt_ids"):
        _Step(True).step(prompt_lengths=LENGTHS)
