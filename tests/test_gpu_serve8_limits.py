"""The 8-bit serving example at the end of a session's table: the step is refused with its reason, and nothing has changed."""
import pytest
import torch

import test_gpu_serve8 as t

pytestmark = pytest.mark.gpu


def test_a_session_longer_than_its_table():
    m, s = t.server("tiny", 2)            # tables of 256 positions
    ids = m.synth.prompt_ids(512, 250, seed=5).tolist()
    s.step({0: ids})
    state = s.free_state.tolist()
    with pytest.raises(RuntimeError, match="do not fit tables of 256 positions"):
        s.step({0: ids[:7], 1: ids[:3]})
    assert s.free_state.tolist() == state and s.length == [250, 0]
    assert torch.isfinite(s.step({0: ids[:6]})[0]).all()
