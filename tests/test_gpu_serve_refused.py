"""The serving example where the pages run out: a request that gets none gives
no tokens, and goes on where it was."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    path = Path(__file__).resolve().parents[1] / "examples" / "serve_q4_kv8.py"
    spec = importlib.util.spec_from_file_location("serve_q4_kv8", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_request_without_pages_gives_no_tokens(example):
    from ztensor_amd.engine import ROCmEngine

    engine = ROCmEngine(stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    prompts, steps = [[5, 6, 7], list(range(100, 230)), list(range(300, 364))], 5
    # 1 + 3 + 1 pages of 64 for the prompts: the last request's next token needs another, the others' do not
    _, server, tokens = example.generate(engine, prompts, steps, pages=5)
    assert server.lens.tolist() == [7, 134, 64] and int(server.free_count) == 0
    assert (tokens[:2] >= 0).all() and tokens[2, 0] >= 0 and (tokens[2, 1:] == -1).all()
    with torch.cuda.stream(engine.stream):
        server.release(1)
        server.step(tokens[:, 0].contiguous(), torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda"), 1, 256)
        torch.cuda.synchronize()
    assert server.took.tolist() == [True, True, True] and server.lens.tolist() == [8, 0, 65]


def test_prompts_without_pages_are_refused(example):
    from ztensor_amd.engine import ROCmEngine

    engine = ROCmEngine(stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="do not hold the prompts"):
        example.generate(engine, [[5, 6, 7], list(range(100))], 2, pages=2)
