"""The example of an 8-bit history and of beams runs."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_runs(capsys):
    from examples import q8_history

    q8_history.main(["--batch", "4", "--prompt", "300", "--steps", "3", "--beams", "2"])
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 4 and "2 x 2 beams" in lines[2] and "int8 history" in lines[3]


def test_beams_of_a_step_continue_the_rows_that_were_chosen():
    from examples import q8_history

    model = q8_history.build("small")
    prompt = torch.randint(0, 32000, (2, 40), generator=torch.Generator().manual_seed(1)).cuda()
    out = q8_history.decode(model, prompt, 6, beams=3)[0]
    assert out.shape == (6, 11)
    assert torch.equal(out.view(2, 3, -1), model.generate_beam(prompt, 3, 11).sequences[..., 40:])
