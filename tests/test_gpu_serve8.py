"""The 8-bit serving example: the operators together. A session's logits do not depend on who else is served or on what its
pages held before."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("serve_8bit", os.path.join(ROOT, "examples", "serve_8bit.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def server(name, sessions, pages=60, layers=2):
    m = example()
    return m, m.Server(m.synth.CONFIGS[name], layers, sessions, pages, ctx=256, seed=3)


def off(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("name", ["tiny", "gqa7", "hd128"])
def test_sessions_together_and_alone(name):
    """Rounded to bfloat16 at every step, values that differ in a last place spread: 2^-8 at each of some 20 roundings on
    the way, which add up as the root of their number, stay below 4 x 2^-8 of the logits' size."""
    m, both = server(name, 3)
    vocab = m.synth.CONFIGS[name]["vocab"]
    prompts = {s: m.synth.prompt_ids(vocab, n, seed=s).tolist() for s, n in ((0, 5), (1, 70), (2, 33))}
    together = both.step(prompts)
    _, alone = server(name, 1)
    for s in prompts:
        got = alone.step({0: prompts[s]})[0]
        assert off(got, together[s]) < 2.0**-6
        alone.end(0)  # (the next session takes over these pages)
    then = both.step({0: [7], 2: [9]})
    assert set(then) == {0, 2}
    got = alone.step({0: prompts[2]})
    got = alone.step({0: [9]})[0]
    assert off(got, then[2]) < 2.0**-6


def test_cut_back_and_fed_again():
    m, s = server("tiny", 2)
    ids = m.synth.prompt_ids(512, 40, seed=5).tolist()
    s.step({0: ids[:32], 1: ids[:9]})
    first = s.step({0: ids[32:]})[0]
    s.step({0: [3, 4, 5, 6, 7, 8, 9, 10, 11]})
    s.cut(0, 32)                       # a page boundary: the pages kept are as they were, and the step is the same
    again = s.step({0: ids[32:]})[0]
    assert torch.equal(again, first)
    head, tail = s.free_state.tolist()
    assert tail - head == 60 - 3 - 1
    s.end(0)
    s.end(1)
    head, tail = s.free_state.tolist()
    assert tail - head == 60


def test_out_of_pages_leaves_the_server_as_it_was():
    m, s = server("tiny", 2, pages=4)
    ids = m.synth.prompt_ids(512, 40, seed=5).tolist()
    want = s.step({0: ids})[0]
    with pytest.raises(RuntimeError, match="1 missing"):
        s.step({1: ids[:30]})
    s.cut(0, 0)
    assert torch.equal(s.step({0: ids})[0], want)
