"""The serving example: its steps, some of them replayed from a graph, leave the
same cache and hidden states as one pass over the whole text."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_steps_are_the_whole_text():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from ztensor_amd.engine import ROCmEngine

    path = Path(__file__).resolve().parents[1] / "examples" / "serve_q4_kv8.py"
    spec = importlib.util.spec_from_file_location("serve_q4_kv8", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    engine = ROCmEngine(stream=torch.cuda.Stream())
    prompts, steps = [[5, 6, 7], list(range(100, 230)), list(range(300, 364))], 6
    torch.cuda.synchronize()
    model, server, tokens = example.generate(engine, prompts, steps)
    assert server.lens.tolist() == [len(p) + steps - 1 for p in prompts]
    used = sum(-(-n // 64) for n in server.lens.tolist())
    assert int(server.free_count) == 64 - used
    with torch.cuda.stream(engine.stream):
        text = [p + t for p, t in zip(prompts, tokens[:, :-1].tolist())]
        new = torch.tensor([len(t) for t in text], dtype=torch.int32, device="cuda")
        # the last token of each once more onto the steps' cache, and the whole text onto an empty one
        server.lens -= 1
        one, _ = server.step(tokens[:, -2].contiguous(), torch.ones_like(new), 1, 256)
        other = example.Server(model, 3)
        whole, plan = other.step(torch.tensor(sum(text, []), device="cuda"), new, 256, 256)
        want = whole[plan.q_start[1:].long() - 1]
        torch.cuda.synchronize()
        # the cache holds 8 bits: steps that round a page more than once differ by some of its steps (1/254 of a page's largest)
        assert float((one - want).norm() / want.norm()) < 0.03
        server.release(1)
        assert int(server.free_count) == 64 - used + 3 and server.lens.tolist()[1] == 0
