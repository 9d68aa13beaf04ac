"""The 8-bit serving example with a shared beginning: norm, rotary positions, attention behind a prefix, and the choice of tokens together
with plan, append and the products, as a server uses them."""
import math

import pytest
import torch

import test_gpu_serve8 as t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["tiny", "gqa7", "hd128"])
@pytest.mark.parametrize("n", [5, 16, 77])
def test_behind_a_shared_beginning_and_with_a_copy_of_it(name, n):
    """Rounded to bfloat16 at every step, as sessions together and alone are (see there): below 4 x 2^-8 of the logits' size. A session's
    pages begin where its own tokens do, so K and V are quantized with other neighbours, too: a step of 2^-8 of a page's largest value
    at most each, of which an output averages many. Twice the bound."""
    m, shared = t.server(name, 3)
    _, copies = t.server(name, 3)
    vocab = m.synth.CONFIGS[name]["vocab"]
    system = m.synth.prompt_ids(vocab, n, seed=9).tolist()
    prompts = {s: m.synth.prompt_ids(vocab, k, seed=s).tolist() for s, k in ((0, 5), (1, 70), (2, 33))}
    shared.share(system)
    got, want = shared.step(prompts), copies.step({s: system + ids for s, ids in prompts.items()})
    for s in prompts:
        assert t.off(got[s], want[s]) < 2.0**-5
    got, want = shared.step({0: [7], 2: [9]}), copies.step({0: [7], 2: [9]})
    assert set(got) == {0, 2}
    for s in got:
        assert t.off(got[s], want[s]) < 2.0**-5
    pages = lambda server: 60 - (server.free_state[1] - server.free_state[0]).item()
    own = [5 + 1, 70, 33 + 1]
    assert pages(shared) == -(-n // 16) + sum(-(-k // 16) for k in own) and pages(copies) == sum(-(-(n + k) // 16) for k in own)


def test_cut_back_behind_a_shared_beginning():
    m, s = t.server("tiny", 2)
    s.share(m.synth.prompt_ids(512, 40, seed=1).tolist())
    ids = m.synth.prompt_ids(512, 40, seed=5).tolist()
    s.step({0: ids[:32], 1: ids[:9]})
    first = s.step({0: ids[32:]})[0]
    s.step({0: [3, 4, 5, 6, 7, 8, 9, 10, 11]})
    s.cut(0, 32)
    assert torch.equal(s.step({0: ids[32:]})[0], first)
    with pytest.raises(RuntimeError, match="before the first step"):
        s.share([1])


def test_tokens_chosen_with_penalties_and_a_mask():
    m = t.example()
    rows = torch.zeros(3, 100, device="cuda")
    rows[:, 40], rows[:, 50], rows[:, 60] = 3.0, 2.9, 2.0
    assert m.choose(rows.clone(), [[1], [40, 40], [40, 2, 50]], repetition=1.2) == [40, 50, 40]   # 3 / 1.2 = 2.5, 2.9 / 1.2 below it
    assert m.choose(rows.clone(), [[1], [40, 40], [40, 2, 50]], repetition=2.0) == [40, 50, 60]
    allowed = torch.zeros(100, dtype=torch.bool, device="cuda")
    allowed[[50, 60, 99]] = True
    got = rows.clone()
    assert m.choose(got, [[1], [50], [60]], repetition=2.0, allowed=allowed) == [50, 60, 50]
    assert (got[:, ~allowed] == -math.inf).all()


def test_a_run(capsys, monkeypatch):
    m = t.example()
    monkeypatch.setattr("sys.argv", ["serve_8bit.py", "--model", "tiny", "--layers", "2", "--sessions", "3", "--steps", "6", "--system", "50"])
    m.main()
    text = capsys.readouterr().out
    assert "session 2" in text and "ms per step" in text
